"""Attention over the 8-bit cache with one key far above all others and tens of thousands of keys far below it, whose weights count
by their number only.

The rows are laid into the cache directly: q and K have a single dimension that counts, K's codes are 0 (so that what is lost of one
weight is lost of all) or -2 .. 2, and 120 at one key (the peak); V's codes are of one sign.  T is the share of all keys but the peak
in the sum of weights, S the largest |score|, u = 2^-24.
Tolerances: a weight is off by at most w = (8 S + 16) u relatively (q to 2^-23, six roundings of a score, exponential, weight to
2^-23); 32-bit sums over L keys, a block of 32 at a time by four waves at least, by (L / 64 + 64) u of the largest partial sum, once
for the outputs and once for the sum of weights.  So, v the largest |V| of the others and p that of the peak:
  |error| <= v T (2 w + (L / 64 + 64) u) + p (T w + (L / 64 + 64) u) + 32 2^-39 v
(the last term is for the 31 keys of the peak's own block: a block's weights are f16 pairs on a scale on which its largest is at
least 2^14, and f16's smallest step is 2^-24, so each is off by up to 2^-25 2^-14 of the peak's), and for prompts, whose weights go
into the matrix instructions on a fixed scale, in steps of 2^-33 of the largest at the coarsest, L 2^-34 v more."""
import numpy as np
import pytest

import batch_model as BM
from ronn_amd.kvcache import PagedKVCache
from test_gpu_batch import Rig

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
GAPS = (20.0, 22.7, 24.2, 25.2, 26.1, 28.55, 29.9, 30.1, 32.3, 35.0, 38.4, 41.0)     # of the peak above the others, powers of two


def page_bytes(codes, which, hd):
    """[blocks, 32, hd] uint8 in the order of a page."""
    n = len(codes)
    if which == 0:
        return codes.reshape(n, 2, 16, hd // 64, 2, 4, 8).transpose(0, 1, 3, 5, 2, 4, 6).reshape(n, -1)
    return codes.reshape(n, 2, 4, 4, hd // 32, 2, 16).transpose(0, 4, 2, 6, 5, 1, 3).reshape(n, -1)


def peaked_row(ctx, kv_heads, hd, fmt, held, new, capacity, peak, peak_v, spread, seed):
    """A cache of one row with `held` + `new` positions, planned for the new ones; K (the dimension that counts) and V [total, hd]."""
    rng = np.random.default_rng(seed)
    total = held + new
    n_b, full = BM.blocks(total), total // 32
    cache = PagedKVCache(ctx, 1, kv_heads, hd, 1, n_b, 32 * n_b, capacity, fmt)
    k = np.zeros((32 * n_b, hd))
    k[:, 0] = rng.integers(-spread, spread + 1, 32 * n_b)
    v = rng.integers(4, 16, (32 * n_b, hd)).astype(np.float64)
    k[peak, 0], v[peak] = 120.0, peak_v
    scale = (1.0, 1.0 / 16)
    for which, x in enumerate((k, v)):
        if fmt == "i8":
            raw = x.astype(np.int8).view(np.uint8)
        else:
            values = BM.e4m3_values()
            order = np.argsort(values[:127])
            at = order[np.searchsorted(values[:127][order], np.abs(x))]
            raw = (at | np.where(x < 0, 128, 0)).astype(np.uint8)
            assert (values[raw] == x).all()
        pages = np.repeat(page_bytes(raw.reshape(n_b, 32, hd), which, hd)[:, None], kv_heads, axis=1)
        cache.buffers[0][which].upload(pages)
        opened = np.zeros((kv_heads, 32, hd), np.float16)
        opened[:, :total - 32 * full] = (x * scale[which])[32 * full:total]
        cache.buffers[0][2 + which].upload(opened)
        cache.buffers[0][4 + which].upload(np.full((n_b, kv_heads), scale[which], np.float32))
    held_b = BM.blocks(held)
    cache.d_table.upload(np.where(np.arange(n_b) < held_b, np.arange(n_b), -1).astype(np.int32))
    cache.d_len.upload(np.array([held], np.int32))
    cache.d_ring_state.upload(np.array([held_b % n_b, n_b - held_b], np.int32))
    cache.plan(ctx.to_device(np.array([new], np.int32)))
    return cache, k[:total, 0], v[:total] / 16


def check_peaked(ctx, kv_heads, group, hd, fmt, held, new, capacity, hint, peak, peak_v, spread, on_a_scale):
    cache, k, v = peaked_row(ctx, kv_heads, hd, fmt, held, new, capacity, peak, peak_v, spread, seed=held + new)
    heads, total = kv_heads * group, held + new
    gap = np.array([GAPS[h % len(GAPS)] for h in range(heads)])
    q = np.zeros((capacity, heads, hd), np.float32)
    q[:, :, 0] = gap * np.log(2) * np.sqrt(hd) / 120
    d_q, d_out = ctx.to_device(q), ctx.alloc(q.nbytes)
    cache.attend(0, d_q, heads, hint, d_out)
    out = d_out.download(np.float32, q.size).reshape(q.shape)
    assert ctx.device_flags() == 0
    others = np.arange(total) != peak
    v_others, v_peak = v[others].max(), np.abs(v[peak]).max()
    for h in range(heads):
        s = q[0, h, 0].astype(np.float64) * k / np.sqrt(hd)
        p = np.exp(s - s.max())
        num = p[:held] @ v[:held]
        den, tail = p[:held].sum(), p[:held][others[:held]].sum()
        for i in range(new):
            num = num + p[held + i] * v[held + i]
            den += p[held + i]
            tail += p[held + i]
            share = tail / den
            w, sums = (8 * np.abs(s).max() + 16) * U, (total / 64 + 64) * U
            bound = v_others * share * (2 * w + sums) + v_peak * (share * w + sums)
            bound += 32 * 2.0 ** -39 * v_others
            bound += total * 2.0 ** -34 * v_others if on_a_scale else 0.0
            off = np.abs(out[i, h] - num / den).max()
            assert off <= bound, (h, gap[h], i, off, bound, (num / den).max())


# unshared (so many tokens could come that nothing is shared) and shared; whole blocks and an unfinished one
@pytest.mark.parametrize("kv_heads,group,hd,fmt,held,capacity", [
    (12, 1, 64, "i8", 16383, 300), (12, 1, 128, "e4m3", 16400, 300), (2, 12, 128, "i8", 16383, 1100), (1, 12, 64, "e4m3", 40001, 1),
    (1, 12, 64, "i8", 131000, 1)])
@pytest.mark.parametrize("peak_v", [0, 15])
@pytest.mark.parametrize("spread", [0, 2])
@pytest.mark.parametrize("late", [False, True])
def test_small_weights_of_a_decode_step(ctx, kv_heads, group, hd, fmt, held, capacity, peak_v, spread, late):
    check_peaked(ctx, kv_heads, group, hd, fmt, held, 1, capacity, 1, held - 100 if late else 0, peak_v, spread, False)


@pytest.mark.parametrize("kv_heads,group,hd,fmt,held,new", [(12, 1, 64, "i8", 20000, 3), (3, 4, 128, "i8", 30005, 4), (4, 3, 64, "e4m3", 50000, 2)])
@pytest.mark.parametrize("peak_v", [0, 15])
@pytest.mark.parametrize("spread", [0, 2])
def test_small_weights_of_a_few_tokens(ctx, kv_heads, group, hd, fmt, held, new, peak_v, spread):
    check_peaked(ctx, kv_heads, group, hd, fmt, held, new, new, 3, 7, peak_v, spread, False)


@pytest.mark.parametrize("kv_heads,group,hd,fmt,held,new", [(12, 1, 64, "i8", 17000, 33), (3, 4, 128, "e4m3", 30000, 50), (1, 12, 64, "i8", 131072, 30)])
@pytest.mark.parametrize("peak_v", [0, 15])
@pytest.mark.parametrize("spread", [0, 2])
@pytest.mark.parametrize("late", [False, True])
def test_small_weights_of_a_prompt(ctx, kv_heads, group, hd, fmt, held, new, peak_v, spread, late):
    check_peaked(ctx, kv_heads, group, hd, fmt, held, new, 64, 50, held - 100 if late else 0, peak_v, spread, True)


@pytest.mark.parametrize("hd,fmt", [(64, "i8"), (128, "e4m3")])
@pytest.mark.parametrize("new,hint", [([1, 1], 1), ([3, 2], 3), ([40, 33], 40)])
def test_scores_whose_units_are_coarse(ctx, hd, fmt, new, hint):
    """Scores from 1e5 to 1e36, where f32 has no bits left for a power of two to be taken off: every output is finite, and where the
    largest score stands clear of the others by more than they can be off, (hd + 8) u sum|q k| / sqrt(hd) each, it is V of that key."""
    rig = Rig(ctx, 4, 2, hd, fmt, rows=2, max_tokens=512, seed=hd)
    rig.step([300, 130])
    q = rig.step(new)
    k, v = zip(*(rig.device_values(r) for r in range(2)))
    clear = 0
    for factor in (1e5, 3e6, 2e7, 1e8, 7e8, 1e10, 1e13, 1e20, 1e35):
        big = (q * np.float32(factor)).astype(np.float32)
        rig.d_q.upload(big)
        out = rig.attend(big, hint)
        assert np.isfinite(out).all(), factor
        for i in range(len(q)):
            r, n = rig.token_row[i], rig.token_pos[i] + 1
            for h in range(4):
                kh, vh = k[r][:n, h // 2], v[r][:n, h // 2]
                s = kh @ big[i, h].astype(np.float64) / np.sqrt(hd)
                off = (hd + 8) * U * (np.abs(kh) @ np.abs(big[i, h]).astype(np.float64)).max() / np.sqrt(hd)
                best = int(s.argmax())
                # 32 below the largest by then, all others together weigh less than n e^-32
                if s[best] - np.partition(s, -2)[-2] > 2 * off + 32:
                    clear += 1
                    assert np.abs(out[i, h] - vh[best]).max() <= 8 * U * np.abs(vh).max() + n * np.exp(-32) * 2 * np.abs(vh).max(), (factor, i, h)
    assert clear > 20 * len(q)
