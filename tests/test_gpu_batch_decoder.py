"""BatchDecoder: the batched operators together as they are used, against a numpy model that runs every sequence by itself
(decoder_model's BitLinears, batch_model's cache and attention).

As for the single decoder, int8 activation codes may fall to the neighbour where a value sits on a rounding boundary, and
here codes of the cache as well; logits are held to the same share of their spread (0.05) as in the single decoder's test.
"""
import numpy as np
import pytest

import batch_model as BM
import decoder_model as DM
from ronn_amd.decoder import BatchDecoder, BitNetDecoder, DecoderConfig

pytestmark = pytest.mark.gpu


class Model:
    """One sequence, called like the device: what the cache holds follows from its tokens, attention of a call sees the
    cache as it is after the call's own tokens."""

    def __init__(self, cfg, lin, w, fmt):
        self.cfg, self.lin, self.w = cfg, lin, w
        self.cache = [BM.Cache(1, cfg.kv_heads, cfg.head_dim, fmt) for _ in range(cfg.layers)]
        self.pos = 0

    def forward(self, tokens):
        """Logits of every token."""
        cfg, w = self.cfg, self.w
        M, heads, kvh, hd = len(tokens), cfg.heads, cfg.kv_heads, cfg.head_dim
        pos = np.arange(self.pos, self.pos + M)
        x = w["embed"][np.asarray(tokens)].astype(np.float32)
        for i in range(cfg.layers):
            p = "L%d." % i
            _, q, s, _ = DM.rmsnorm_quant(x, w[p + "g_attn"], cfg.eps)
            qkv = self.lin[p + "wqkv"](q, s).reshape(M, heads + 2 * kvh, hd)
            qr = BM.rope64(qkv[:, :heads], pos, cfg.rope_theta)
            self.cache[i].append(0, BM.rope64(qkv[:, heads:heads + kvh], pos, cfg.rope_theta), qkv[:, heads + kvh:])
            att = BM.attention(qr, pos, *self.cache[i].values(0)).astype(np.float32)
            _, q, s, _ = DM.rmsnorm_quant(att.reshape(M, -1), w[p + "g_attn_sub"], cfg.eps)
            x = (x + self.lin[p + "wo"](q, s)).astype(np.float32)
            _, q, s, _ = DM.rmsnorm_quant(x, w[p + "g_ffn"], cfg.eps)
            gu = self.lin[p + "wgu"](q, s)
            g, u = gu[:, :cfg.ffn], gu[:, cfg.ffn:]
            _, q, s, _ = DM.rmsnorm_quant(((g / (1.0 + np.exp(-g))) * u).astype(np.float32), w[p + "g_ffn_sub"], cfg.eps)
            x = (x + self.lin[p + "wdown"](q, s)).astype(np.float32)
        _, q, s, _ = DM.rmsnorm_quant(x, w["g_final"], cfg.eps)
        self.pos += M
        return self.lin["lm_head"](q, s)


def build(ctx, kv_heads, seed, max_seq=160):
    cfg = DecoderConfig(layers=2, hidden=256, heads=2, head_dim=128, ffn=384, vocab=1000, max_seq=max_seq, kv_heads=kv_heads)
    w = DM.random_weights(cfg, seed)
    dec = BitNetDecoder(ctx, cfg, max_batch_tokens=16)
    dec.load_weights(w)
    lin = {k: DM.Linear(v) for k, v in w.items() if v.ndim == 2 and k != "embed"}
    return cfg, w, dec, lin


def agree(next_token, logits):
    """NextToken against the model's logits: the alternatives are its largest, log probabilities and entropy follow."""
    lp, ent, tok, top_lp = BM.logprobs(logits[None].astype(np.float32), [-1], len(next_token.top_tokens))
    spread = logits.std()
    mine = logits - logits.max()
    mine = mine - np.log(np.exp(mine.astype(np.float64)).sum())
    # every alternative has the log probability that the model gives it, and none of the model's is missed by more
    assert np.abs(next_token.top_logprobs - mine[next_token.top_tokens]).max() < 0.06 * spread
    assert np.abs(np.sort(next_token.top_logprobs)[::-1] - top_lp[0]).max() < 0.06 * spread
    assert (np.diff(next_token.top_logprobs) <= 0).all() and len(set(next_token.top_tokens)) == len(next_token.top_tokens)
    assert next_token.token == next_token.top_tokens[0] and next_token.logprob == next_token.top_logprobs[0]
    assert abs(next_token.entropy - ent[0]) < 0.06 * spread


@pytest.mark.parametrize("kv_heads,fmt", [(2, "i8"), (1, "e4m3")])
def test_sequences_come_and_go(ctx, kv_heads, fmt):
    cfg, w, dec, lin = build(ctx, kv_heads, seed=3)
    bat = BatchDecoder(dec, rows=4, pages=12, max_tokens=96, fmt=fmt, top=4)
    rng = np.random.default_rng(1)
    models = {}

    def start(prompts):
        got = bat.start(prompts)
        for r, ids in prompts.items():
            models[r] = Model(cfg, lin, w, fmt)
            agree(got[r], models[r].forward(ids)[-1])

    def step(n):
        for _ in range(n):
            tokens = {r: t.token for r, t in bat.running.items()}
            got = bat.step()
            assert sorted(got) == sorted(tokens)
            for r, t in tokens.items():
                agree(got[r], models[r].forward([t])[-1])

    start({0: rng.integers(0, 1000, 11), 2: rng.integers(0, 1000, 45)})
    step(3)
    start({1: rng.integers(0, 1000, 31)})
    step(3)                                   # row 1 completes its first block here
    bat.finish(0)
    step(1)
    start({0: rng.integers(0, 1000, 64), 3: [7]})
    step(2)
    bat.finish([2, 1])
    step(1)
    bat.finish([0, 3])
    assert bat.cache.free_pages() == 12 and (bat.cache.lengths() == 0).all() and not bat.running
    assert ctx.device_flags() == 0
    bat.close()


def test_graph_steps_equal_eager_steps(ctx):
    cfg, w, dec, lin = build(ctx, 1, seed=4)
    rng = np.random.default_rng(2)
    prompts = {0: rng.integers(0, 1000, 30), 1: rng.integers(0, 1000, 5), 2: rng.integers(0, 1000, 63)}
    runs = []
    for graph in (True, False):
        bat = BatchDecoder(dec, rows=3, max_tokens=128, top=2)
        bat.start(prompts)
        seen = []
        for i in range(8):
            got = bat.step(use_graph=graph)
            seen += [(r, t.token, t.logprob, t.entropy, tuple(t.top_tokens), tuple(t.top_logprobs)) for r, t in sorted(got.items())]
            if i == 3:
                bat.finish(1)                    # another number of rows: another captured step
            if i == 5:
                bat.start({1: prompts[1]})       # and the first one again
        runs.append(seen)
        bat.close()
    assert runs[0] == runs[1]


def test_score(ctx):
    cfg, w, dec, lin = build(ctx, 2, seed=5, max_seq=512)
    bat = BatchDecoder(dec, rows=3, max_tokens=400)          # 378 tokens: two rounds of logits
    rng = np.random.default_rng(3)
    prompts = {0: rng.integers(0, 1000, 77), 2: rng.integers(0, 1000, 300), 1: np.array([5])}
    got = bat.score(prompts)
    assert sorted(got) == [0, 1, 2] and got[1][0].size == 0
    for r in (0, 2):
        ids = prompts[r]
        logits = Model(cfg, lin, w, "i8").forward(ids)[:-1]
        lp, ent, _, _ = BM.logprobs(logits.astype(np.float32), ids[1:], 0)
        assert got[r][0].shape == got[r][1].shape == (ids.size - 1,)
        assert np.abs(got[r][0] - lp).max() < 0.08 * logits.std() and np.abs(got[r][1] - ent).max() < 0.08 * logits.std()
        assert abs(got[r][0].mean() - lp.mean()) < 0.005 * logits.std()
    assert bat.cache.free_pages() == bat.cache.pages and not bat.running
    # the rows are free again and the state is clean: the same scores
    again = bat.score(prompts)
    assert all((again[r][0] == got[r][0]).all() and (again[r][1] == got[r][1]).all() for r in got)


def test_refusals_leave_the_state_alone(ctx):
    cfg, w, dec, lin = build(ctx, 1, seed=6, max_seq=64)
    with pytest.raises(ValueError, match="BatchDecoder"):
        dec.prefill(np.arange(5))
    for kw in (dict(rows=0), dict(rows=4, max_tokens=3), dict(rows=2, top=0), dict(rows=2, top=33), dict(rows=2, fmt="i4")):
        with pytest.raises(ValueError):
            BatchDecoder(dec, **kw)
    bat = BatchDecoder(dec, rows=3, pages=3, max_tokens=96)
    for bad in ({}, {3: [1]}, {-1: [1]}, {0: []}, {0: [[1, 2]]}, {0: np.arange(65)}, {0: np.arange(60), 1: np.arange(40)},
                {0: np.arange(40), 1: np.arange(40)}):
        with pytest.raises(ValueError):
            bat.start(bad)
    with pytest.raises(ValueError, match="no row"):
        bat.step()
    with pytest.raises(ValueError):
        bat.finish(0)
    bat.start({0: np.arange(62), 2: np.arange(32)})
    for bad in ({0: [1]}, {1: [5]}):             # row 0 runs; no page is left
        with pytest.raises(ValueError):
            bat.start(bad)
    with pytest.raises(ValueError, match="pages"):
        bat.step()                               # row 2 would need a fourth page
    bat.finish(2)
    bat.step()
    bat.step()
    with pytest.raises(ValueError, match="max_seq"):
        bat.step()
    assert list(bat.cache.lengths()) == [64, 0, 0] and ctx.device_flags() == 0
    bat.finish([0])
    assert bat.cache.free_pages() == 3
    with pytest.raises(ValueError):
        DecoderConfig(heads=6, kv_heads=4)
    bat.close()


def test_full_size_batch(ctx):
    """The decoder's default configuration with five K/V heads, 16 ragged prompts of up to 512 tokens: graph and eager
    steps give the same bits, everything is finite, sequences differ."""
    cfg = DecoderConfig(max_seq=600, kv_heads=5)
    dec = BitNetDecoder(ctx, cfg, max_batch_tokens=16)
    dec.init_random(seed=4)
    rng = np.random.default_rng(7)
    prompts = {r: rng.integers(0, cfg.vocab, 1 + (r * 97) % 512) for r in range(16)}
    runs = []
    for graph in (True, False):
        print("full-size batch, graph =", graph, flush=True)
        bat = BatchDecoder(dec, rows=16, max_tokens=sum(p.size for p in prompts.values()), top=5)
        bat.start(prompts)
        seen = [bat.step(use_graph=graph) for _ in range(6)]
        runs.append([(r, t.token, t.logprob, t.entropy) for got in seen for r, t in sorted(got.items())])
        assert all(np.isfinite([t.logprob, t.entropy]).all() for got in seen for t in got.values())
        bat.close()
        del bat
    assert runs[0] == runs[1] and len({t for _, t, _, _ in runs[0]}) > 8
    assert ctx.device_flags() == 0
