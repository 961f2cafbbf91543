"""Top alternatives where a workgroup takes a row, or its part of one, in several sweeps (more than 512 / rows < vocab / 8192) and a
later sweep has more candidates than its list holds: equal logits behind lower ones, logits of few distinct values, ascending rows."""
import numpy as np
import pytest

from test_gpu_batch import check_logprobs

pytestmark = pytest.mark.gpu


def pattern(kind, vocab, rng):
    """A row whose first 8192 logits lie below the rest."""
    x = np.empty(vocab, np.float32)
    front, back = x[:8192], x[8192:]
    if kind == "equals apart":                   # the largest, with lower ones between them
        front[:], back[:] = 0.0, 0.5
        back[::int(rng.integers(20, 60))] = 1.0
    elif kind == "every second":
        x[:] = -50.0
        back[::2] = 1.0
    elif kind == "clipped":                      # a masked front, the rest clipped at a cap
        front[:] = -np.inf
        back[:] = np.minimum(rng.normal(0, 1, back.size), 1.0)
    elif kind == "coarse":                       # values of 8-bit resolution
        front[:] = -1e9
        back[:] = np.round(rng.normal(0, 1, back.size) * 16) / 16
    elif kind == "masked":                       # one value, a third of it masked
        front[:] = rng.normal(-30, 1, front.size)
        back[:] = np.where(rng.random(back.size) < 0.3, -np.inf, 2.0)
    elif kind == "held ones count":              # the front holds a few of the same largest value, and one above
        front[:], back[:] = 0.0, 0.5
        front[[5, 8000]] = 1.0
        front[17] = 1.5
        back[1::35] = 1.0
    elif kind == "bound stays":                  # ... or all that can count
        front[:], back[:] = 0.0, -1.0
        front[100:200] = 1.0
        back[::3] = 1.0
    elif kind == "few above equals":             # some above the equals, all of them late
        front[:], back[:] = -2.0, 0.0
        back[::3] = 1.0
        back[-40::9] = 1.25 + np.arange(len(back[-40::9]), dtype=np.float32) / 64
    elif kind == "ascending":
        x[:] = np.arange(vocab, dtype=np.float32) / vocab * 30
    elif kind == "ascending in steps":
        x[:] = np.floor(np.arange(vocab, dtype=np.float32) / 3000)
    elif kind == "nan":                          # NaN among them, as many as numbers that count
        front[:], back[:] = -5.0, 0.0
        back[::4] = np.nan
        back[1::4] = 1.0
    return x


KINDS = ["equals apart", "every second", "clipped", "coarse", "masked", "held ones count", "bound stays", "few above equals",
         "ascending", "ascending in steps", "nan"]


# (rows, vocab): a workgroup for a row of two sweeps, of a bit more, of five; two or three for a row; many for a single long one
@pytest.mark.parametrize("rows,vocab", [(600, 16384), (300, 16391), (257, 40000), (200, 40000), (100, 60003), (1, 262147)])
@pytest.mark.parametrize("top", [1, 2, 5, 8, 32])
def test_equals_in_a_later_sweep(ctx, rows, vocab, top):
    rng = np.random.default_rng(rows + top)
    for first in range(len(KINDS) if rows == 1 else 1):
        x = np.stack([pattern(KINDS[(first + r) % len(KINDS)], vocab, rng) for r in range(min(rows, 2 * len(KINDS)))])
        x = x[np.arange(rows) % len(x)]
        check_logprobs(ctx, x, rng.integers(0, vocab, rows), top)


@pytest.mark.parametrize("rows,vocab", [(300, 9000), (300, 50021), (180, 50021)])
@pytest.mark.parametrize("mask", [-np.inf, -1e9, 0.0])
def test_masked_rows_in_several_sweeps(ctx, rows, vocab, mask):
    """Nearly all logits at one value; smaller ones at the front, NaN among them, in pieces at any 4-byte address."""
    rng = np.random.default_rng(vocab)
    x = np.full((8, vocab), mask, np.float32)
    for r, n in enumerate((0, 1, 5, 19, 20, 300, 40, 6)):
        x[r, rng.choice(vocab, n, replace=False)] = rng.normal(5, 2, n)
    x[6, :8250] = -2e9 if np.isfinite(mask) else mask
    x[7, [3, 4000, 8999]] = np.nan
    x = x[np.arange(rows) % 8]
    check_logprobs(ctx, x, rng.integers(0, vocab, rows), 20)
    check_logprobs(ctx, x[:, :vocab - 3], rng.integers(0, vocab - 3, rows), 32, pitch=vocab + 2, shift=1)
