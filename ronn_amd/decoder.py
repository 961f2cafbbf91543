"""A BitNet-b1.58-style decoder assembled from the library's kernels.

Every linear layer is a ternary BitLinear: RMSNorm, per-token int8 quantisation (one fused
kernel), ternary matmul with the fused dequantisation.  Attention keeps K and V in f16.  The
reference has no decoder (its BitNet provider stops at the matmul,
crates/ronn-providers/src/bitnet/kernels.rs:134-178), so the layer formulas are the usual
LLaMA / BitNet-b1.58 ones; tests/decoder_model.py restates them in numpy.

A decode step is 122 kernel launches; it reads the position and the previous token from
device memory, so it is captured once in a HIP graph and replayed per token.

BitNetDecoder serves one sequence over contiguous f16 caches; BatchDecoder serves several at once
with the same weights over the paged 8-bit cache (kvcache.py), with log probabilities.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import dataclasses
import time

import numpy as np

from . import _lib
from ._lib import check
from .device import Context, DeviceBuffer
from .kvcache import PagedKVCache


class _AsHeads(int):
    """A number of K/V heads that nobody gave: it stays that of the query heads."""


@dataclasses.dataclass
class DecoderConfig:
    layers: int = 24
    hidden: int = 2560
    heads: int = 20
    head_dim: int = 128
    ffn: int = 6912
    vocab: int = 32000
    max_seq: int = 1024
    eps: float = 1e-5
    rope_theta: float = 10000.0
    kv_heads: int = 0       # K/V heads; 0: as many as query heads.  Fewer are served by BatchDecoder only

    def __setattr__(self, name, value):
        if name == "kv_heads" and (not value or isinstance(value, _AsHeads)):
            value = _AsHeads(self.heads)
        object.__setattr__(self, name, value)
        if name == "heads" and isinstance(vars(self).get("kv_heads"), _AsHeads):
            self.kv_heads = 0

    def __post_init__(self):
        if self.kv_heads < 0 or (self.kv_heads and self.heads % self.kv_heads):
            raise ValueError("heads (%d) must be a multiple of kv_heads (%d)" % (self.heads, self.kv_heads))

    @property
    def attn_dim(self) -> int:
        return self.heads * self.head_dim

    @property
    def qkv_dim(self) -> int:
        return (self.heads + 2 * self.kv_heads) * self.head_dim

    def linear_shapes(self):
        """(name, K, N) of the four BitLinear layers of a block."""
        return (("wqkv", self.hidden, self.qkv_dim), ("wo", self.attn_dim, self.hidden),
                ("wgu", self.hidden, 2 * self.ffn), ("wdown", self.ffn, self.hidden))

    def packed_weight_bytes_per_token(self) -> int:
        per_layer = sum(k * n for _, k, n in self.linear_shapes())
        return (self.layers * per_layer + self.hidden * self.vocab) // 4


class _Linear:
    def __init__(self, tiled: DeviceBuffer, scale: float, K: int, N: int):
        self.tiled, self.scale, self.K, self.N = tiled, float(scale), K, N


class BitNetDecoder:
    """Weights, caches and scratch buffers of one decoder on one GPU."""

    def __init__(self, ctx: Context, cfg: DecoderConfig, max_batch_tokens: int = 512):
        if cfg.head_dim != 128:
            raise ValueError("head_dim must be 128")
        self.ctx, self.cfg, self.lib = ctx, cfg, ctx.lib
        self.max_tokens = max_batch_tokens
        H, A, F, V, T = cfg.hidden, cfg.attn_dim, cfg.ffn, cfg.vocab, max_batch_tokens
        a = ctx.alloc
        self.x = a(4 * T * H)
        self.o = a(4 * T * H)
        self.d = a(4 * T * H)
        self.qkv = a(4 * T * cfg.qkv_dim)
        self.att = a(4 * T * A)
        self.gu = a(4 * T * 2 * F)
        self.logits = a(4 * V)
        pitch = ctx.act_pitch(max(H, A, F))
        self.acts = (a(T * pitch), a(4 * T), a(4 * T))
        self.tokens = a(4 * T)
        self.pos = a(4)
        self.history = a(4 * cfg.max_seq)
        # the f16 caches; grouped K/V heads have none (BatchDecoder brings its own)
        cache = 2 * cfg.heads * cfg.max_seq * cfg.head_dim
        layers = cfg.layers if cfg.kv_heads == cfg.heads else 0
        self.kcache = [a(cache) for _ in range(layers)]
        self.vcache = [a(cache) for _ in range(layers)]
        self.blocks = []
        self.embed = self.g_final = self.lm_head = None
        self._graph = None
        self._pos = 0   # host copy of the device position counter

    # -- weights ---------------------------------------------------------------------------
    def _linear_from_device_f32(self, d_w: DeviceBuffer, K: int, N: int) -> _Linear:
        d_p, scale, _, _ = self.ctx.quantize_ternary(d_w, K * N, _lib.SUM_STRICT_SEQ)
        tiled = self.ctx.tile_weights(d_p, K, N)
        self.ctx.sync()
        d_p.free()
        return _Linear(tiled, scale, K, N)

    def _vector(self, v: np.ndarray) -> DeviceBuffer:
        return self.ctx.to_device(np.ascontiguousarray(v, dtype=np.float32))

    def load_weights(self, w: dict):
        """w: numpy arrays 'embed' [V,H], 'g_final' [H], 'lm_head' [H,V], and per layer i
        'L{i}.g_attn' [H], 'L{i}.wqkv' [H, qkv_dim], 'L{i}.g_attn_sub' [A], 'L{i}.wo' [A,H],
        'L{i}.g_ffn' [H], 'L{i}.wgu' [H,2F], 'L{i}.g_ffn_sub' [F], 'L{i}.wdown' [F,H]."""
        cfg = self.cfg

        def lin(name, K, N):
            arr = np.ascontiguousarray(w[name], dtype=np.float32)
            assert arr.shape == (K, N), (name, arr.shape)
            d_w = self.ctx.to_device(arr)
            out = self._linear_from_device_f32(d_w, K, N)
            d_w.free()
            return out

        self.embed = self._vector(w["embed"])
        self.g_final = self._vector(w["g_final"])
        self.lm_head = lin("lm_head", cfg.hidden, cfg.vocab)
        self.blocks = []
        for i in range(cfg.layers):
            b = {"g_attn": self._vector(w["L%d.g_attn" % i]),
                 "g_attn_sub": self._vector(w["L%d.g_attn_sub" % i]),
                 "g_ffn": self._vector(w["L%d.g_ffn" % i]),
                 "g_ffn_sub": self._vector(w["L%d.g_ffn_sub" % i])}
            for name, K, N in cfg.linear_shapes():
                b[name] = lin("L%d.%s" % (i, name), K, N)
            self.blocks.append(b)

    def init_random(self, seed: int = 1, sigma: float = 0.02):
        """Random-initialised weights generated on the device (N(0, sigma) linears and
        embedding, unit norm gains)."""
        cfg, ctx = self.cfg, self.ctx
        counter = [seed * 1000]

        def normal(n, s):
            buf = ctx.alloc(4 * n)
            counter[0] += 1
            check(self.lib.rbn_synth_normal_device_f32(ctx.handle, counter[0], s, buf.ptr, n))
            return buf

        def lin(K, N):
            d_w = normal(K * N, sigma)
            out = self._linear_from_device_f32(d_w, K, N)
            d_w.free()
            return out

        ones = lambda n: self._vector(np.ones(n, dtype=np.float32))
        self.embed = normal(cfg.vocab * cfg.hidden, sigma)
        self.g_final = ones(cfg.hidden)
        self.lm_head = lin(cfg.hidden, cfg.vocab)
        self.blocks = []
        for _ in range(cfg.layers):
            b = {"g_attn": ones(cfg.hidden), "g_attn_sub": ones(cfg.attn_dim),
                 "g_ffn": ones(cfg.hidden), "g_ffn_sub": ones(cfg.ffn)}
            for name, K, N in cfg.linear_shapes():
                b[name] = lin(K, N)
            self.blocks.append(b)
        ctx.sync()

    # -- one forward pass over M tokens starting at the position in self.pos -----------------
    def _norm_quant(self, x, delta, gamma: DeviceBuffer, M: int, H: int, row0: int = 0, gate_up=None):
        off = 4 * row0 * H
        check(self.lib.rbn_rmsnorm_quant_i8(
            self.ctx.handle, (x.ptr + off) if x is not None else None,
            (delta.ptr + off) if delta is not None else None,
            gate_up.ptr if gate_up is not None else None, gamma.ptr,
            self.cfg.eps, M, H, self.acts[0].ptr, self.acts[1].ptr, self.acts[2].ptr))

    def _linear(self, lin: _Linear, M: int, out: DeviceBuffer):
        self.ctx.matmul(self.acts, lin.tiled, lin.scale, M, lin.K, lin.N, d_out=out)

    def _bitlinear1(self, lin: _Linear, gamma: DeviceBuffer, out: DeviceBuffer, x=None, gate_up=None,
                    residual=None, row0: int = 0):
        """One token: norm + quant + GEMV (+ residual) in one launch."""
        off = 4 * row0 * lin.K
        check(self.lib.rbn_bitlinear_gemv_f32(
            self.ctx.handle, (x.ptr + off) if x is not None else None,
            gate_up.ptr if gate_up is not None else None, gamma.ptr, self.cfg.eps, lin.tiled.ptr, lin.scale,
            lin.K, lin.N, residual.ptr if residual is not None else None, out.ptr))

    def forward_one(self):
        """forward(1) with five launches per layer: every BitLinear is one kernel, the
        residual additions ride on the o and down projections."""
        cfg, lib, hnd = self.cfg, self.lib, self.ctx.handle
        for i, b in enumerate(self.blocks):
            self._bitlinear1(b["wqkv"], b["g_attn"], self.qkv, x=self.x)
            check(lib.rbn_attention_decode_f16kv(hnd, self.qkv.ptr, self.pos.ptr, cfg.heads, cfg.head_dim,
                                                 cfg.rope_theta, self.kcache[i].ptr, self.vcache[i].ptr,
                                                 cfg.max_seq, self.att.ptr))
            self._bitlinear1(b["wo"], b["g_attn_sub"], self.x, x=self.att, residual=self.x)
            self._bitlinear1(b["wgu"], b["g_ffn"], self.gu, x=self.x)
            self._bitlinear1(b["wdown"], b["g_ffn_sub"], self.x, gate_up=self.gu, residual=self.x)
        self._bitlinear1(self.lm_head, self.g_final, self.logits, x=self.x)
        # position + 1, arg-max, history, and the next step's embedding in one launch
        check(lib.rbn_greedy_next_f32(hnd, self.logits.ptr, cfg.vocab, self.tokens.ptr, self.history.ptr,
                                      self.pos.ptr, cfg.max_seq, self.embed.ptr, cfg.hidden, self.x.ptr))

    def launches_per_token(self) -> int:
        """Kernel launches of one decode step (forward_one)."""
        return 5 * self.cfg.layers + 2

    def forward(self, M: int):
        """Tokens self.tokens[0:M] at positions *pos .. *pos+M-1; leaves the logits of the
        last token in self.logits and its arg-max in self.tokens[0] and the history."""
        cfg, lib, hnd = self.cfg, self.lib, self.ctx.handle
        H, A, F = cfg.hidden, cfg.attn_dim, cfg.ffn
        if M > self.max_tokens:
            raise ValueError("M exceeds max_batch_tokens")
        check(lib.rbn_embed_f32(hnd, self.embed.ptr, self.tokens.ptr, M, H, cfg.vocab, self.x.ptr))
        pending = None
        for i, b in enumerate(self.blocks):
            self._norm_quant(self.x, pending, b["g_attn"], M, H)
            self._linear(b["wqkv"], M, self.qkv)
            if M == 1:
                check(lib.rbn_attention_decode_f16kv(hnd, self.qkv.ptr, self.pos.ptr, cfg.heads, cfg.head_dim,
                                                     cfg.rope_theta, self.kcache[i].ptr, self.vcache[i].ptr,
                                                     cfg.max_seq, self.att.ptr))
            else:
                check(lib.rbn_rope_kv_store_f16(hnd, self.qkv.ptr, self.pos.ptr, M, cfg.heads, cfg.head_dim,
                                                cfg.rope_theta, self.kcache[i].ptr, self.vcache[i].ptr,
                                                cfg.max_seq))
                check(lib.rbn_attention_f16kv(hnd, self.qkv.ptr, self.pos.ptr, M, cfg.heads, cfg.head_dim,
                                              self.kcache[i].ptr, self.vcache[i].ptr, cfg.max_seq,
                                              self.att.ptr))
            self._norm_quant(self.att, None, b["g_attn_sub"], M, A)
            self._linear(b["wo"], M, self.o)
            self._norm_quant(self.x, self.o, b["g_ffn"], M, H)
            self._linear(b["wgu"], M, self.gu)
            self._norm_quant(None, None, b["g_ffn_sub"], M, F, gate_up=self.gu)   # SwiGLU fused in
            self._linear(b["wdown"], M, self.d)
            pending = self.d
        # only the last token needs logits; the pending residual is added for every row, so
        # that self.x is the complete residual stream
        if M > 1:
            self._norm_quant(self.x, pending, self.g_final, M - 1, H)
        self._norm_quant(self.x, pending, self.g_final, 1, H, row0=M - 1)
        self._linear(self.lm_head, 1, self.logits)
        check(lib.rbn_add_i32(hnd, self.pos.ptr, M))
        check(lib.rbn_argmax_f32(hnd, self.logits.ptr, cfg.vocab, self.tokens.ptr, self.history.ptr,
                                 self.pos.ptr, cfg.max_seq))

    # -- generation ------------------------------------------------------------------------
    def reset(self):
        check(self.lib.rbn_fill_u8(self.ctx.handle, self.pos.ptr, 0, 4))
        self._pos = 0

    def prefill(self, prompt: np.ndarray):
        """Runs the prompt from position 0.  The token predicted after it goes to history slot
        len(prompt), so the prompt has to be shorter than max_seq."""
        if self.cfg.kv_heads != self.cfg.heads:
            raise ValueError("a decoder with %d K/V heads for %d query heads is served by BatchDecoder"
                             % (self.cfg.kv_heads, self.cfg.heads))
        prompt = np.ascontiguousarray(prompt, dtype=np.int32)
        if prompt.ndim != 1 or len(prompt) == 0:
            raise ValueError("the prompt must be a non-empty vector of token ids")
        if len(prompt) >= self.cfg.max_seq:
            raise ValueError("a prompt of %d tokens does not fit max_seq = %d (history slot %d is needed)"
                             % (len(prompt), self.cfg.max_seq, len(prompt)))
        self.reset()
        check(self.lib.rbn_h2d(self.ctx.handle, self.tokens.ptr, prompt.ctypes.data, prompt.nbytes))
        self.forward(len(prompt))
        self._pos = len(prompt)

    def capture_decode_step(self):
        if self._graph is None:
            self.ctx.graph_begin()
            self.forward_one()
            self._graph = self.ctx.graph_end()
        return self._graph

    def decode(self, n_tokens: int, use_graph: bool = True):
        """Greedy decoding of n_tokens more tokens; returns (tokens, seconds)."""
        if n_tokens < 0 or self._pos + n_tokens >= self.cfg.max_seq:
            raise ValueError("decoding %d tokens from position %d would pass max_seq = %d"
                             % (n_tokens, self._pos, self.cfg.max_seq))
        g = self.capture_decode_step() if use_graph else None
        # a step expects the embedding of the previous token in self.x (each step leaves the
        # next one's there; after a prompt it has to be looked up once)
        check(self.lib.rbn_embed_f32(self.ctx.handle, self.embed.ptr, self.tokens.ptr, 1, self.cfg.hidden,
                                     self.cfg.vocab, self.x.ptr))
        self.ctx.sync()
        t0 = time.perf_counter()
        for _ in range(n_tokens):
            if g is not None:
                self.ctx.graph_launch(g)
            else:
                self.forward_one()
        self.ctx.sync()
        dt = time.perf_counter() - t0
        self._pos += n_tokens
        return self.generated(n_tokens + 1)[1:], dt

    def generated(self, n: int) -> np.ndarray:
        """The last n generated tokens (history[p] = token predicted for position p)."""
        pos = int(self.pos.download(np.int32, 1)[0])
        hist = self.history.download(np.int32, self.cfg.max_seq)
        return hist[pos - n + 1:pos + 1].copy()

    def last_logits(self) -> np.ndarray:
        return self.logits.download(np.float32, self.cfg.vocab)


@dataclasses.dataclass
class NextToken:
    """What the model says of the token after a row's last one: the greedy choice, its log probability, the
    entropy (nats) of the distribution, and the `top` most probable tokens with their log probabilities."""
    token: int
    logprob: float
    entropy: float
    top_tokens: np.ndarray
    top_logprobs: np.ndarray


class BatchDecoder:
    """Several sequences at once with the weights of a BitNetDecoder, over a paged 8-bit K/V cache.

    A row is the place of one sequence (0 .. rows - 1): start() puts prompts into free rows, step() advances every
    running row by its greedy token, finish() frees rows.  score() gives the log probabilities of given tokens.
    pages: pages of 32 positions shared by the rows (0: enough for every row at cfg.max_seq); max_tokens: the most
    tokens of one call; top: alternatives that come with every token (1 to 32).  A call that is refused changes nothing; where one
    fails on the way (a launch, say), the rows that it had advanced on the device end and are free again.  The decoder does not look at
    ctx.device_flags(): FLAG_KV_NONFINITE there says that since it was read last a key or value was saturated or a NaN made 0."""

    LOGIT_ROWS = 256    # rows of logits computed at a time when prompts are scored

    def __init__(self, dec: BitNetDecoder, rows: int, pages: int = 0, max_tokens: int = 512, fmt: str = "i8", top: int = 1):
        cfg, ctx = dec.cfg, dec.ctx
        if not dec.blocks:
            raise ValueError("the decoder has no weights yet")
        if not 1 <= top <= _lib.TOP_MAX:
            raise ValueError("top must be in [1, %d]" % _lib.TOP_MAX)
        if rows < 1 or max_tokens < rows:
            raise ValueError("max_tokens (%d) must hold one token of each of the %d rows" % (max_tokens, rows))
        self.dec, self.cfg, self.ctx, self.lib = dec, cfg, ctx, ctx.lib
        self.rows, self.max_tokens, self.top = rows, max_tokens, top
        pages = pages or rows * -(-cfg.max_seq // _lib.KV_BLOCK)
        self.cache = PagedKVCache(ctx, cfg.layers, cfg.kv_heads, cfg.head_dim, rows, pages, cfg.max_seq, max_tokens, fmt)
        H, A, F, V, T = cfg.hidden, cfg.attn_dim, cfg.ffn, cfg.vocab, max_tokens
        a = ctx.alloc
        self.x, self.o, self.d = a(4 * T * H), a(4 * T * H), a(4 * T * H)
        self.qkv, self.q, self.att, self.gu = a(4 * T * cfg.qkv_dim), a(4 * T * A), a(4 * T * A), a(4 * T * 2 * F)
        self.pitch = ctx.act_pitch(max(H, A, F))
        self.acts = (a(T * self.pitch), a(4 * T), a(4 * T))
        self.last = (a(rows * self.pitch), a(4 * rows), a(4 * rows))   # the last token of each row, for the logits
        self.tokens, self.targets = a(4 * T), a(4 * max(T, rows))
        self.d_new = a(4 * rows)
        self.logit_rows = max(rows, min(T, self.LOGIT_ROWS))
        R = self.logit_rows
        self.logits = a(4 * R * V)
        # one buffer for what comes back: log probability, entropy, top tokens, top log probabilities
        self.stats = a(4 * R * (2 + 2 * top))
        self._graphs = {}
        self._len = np.zeros(rows, dtype=np.int64)     # host copies of what the device holds
        self._free = pages
        self._next = {}                                # running rows: their NextToken
        self._lost = False                             # whether they can no longer be trusted

    # -- queueing ------------------------------------------------------------------------------------
    def _forward(self, M: int, max_new: int):
        """self.tokens[0:M], planned by self.d_new, through all layers; leaves the quantised, normalised last hidden
        state of every token in self.acts."""
        cfg, dec, cache = self.cfg, self.dec, self.cache
        H, A, F = cfg.hidden, cfg.attn_dim, cfg.ffn
        batch = cache.batch(M)
        cache.plan(self.d_new, batch)
        check(self.lib.rbn_embed_f32(self.ctx.handle, dec.embed.ptr, self.tokens.ptr, M, H, cfg.vocab, self.x.ptr))
        pending = None
        for i, b in enumerate(dec.blocks):
            self._norm_quant(self.x, pending, b["g_attn"], M, H)
            self._linear(b["wqkv"], M, self.qkv)
            cache.store(i, self.qkv, cfg.heads, cfg.rope_theta, self.q, batch)
            cache.attend(i, self.q, cfg.heads, max_new, self.att, batch)
            self._norm_quant(self.att, None, b["g_attn_sub"], M, A)
            self._linear(b["wo"], M, self.o)
            self._norm_quant(self.x, self.o, b["g_ffn"], M, H)
            self._linear(b["wgu"], M, self.gu)
            self._norm_quant(None, None, b["g_ffn_sub"], M, F, gate_up=self.gu)
            self._linear(b["wdown"], M, self.d)
            pending = self.d
        self._norm_quant(self.x, pending, dec.g_final, M, H)

    def _norm_quant(self, x, delta, gamma, M, H, gate_up=None):
        check(self.lib.rbn_rmsnorm_quant_i8(
            self.ctx.handle, x.ptr if x is not None else None, delta.ptr if delta is not None else None,
            gate_up.ptr if gate_up is not None else None, gamma.ptr, self.cfg.eps, M, H, self.acts[0].ptr,
            self.acts[1].ptr, self.acts[2].ptr))

    def _linear(self, lin, M, out):
        self.ctx.matmul(self.acts, lin.tiled, lin.scale, M, lin.K, lin.N, d_out=out)

    def _logprobs(self, acts, row0: int, M: int, with_targets: bool):
        """Logits of rows row0 .. row0 + M of acts, and what self.stats holds of them."""
        head, V, top, R = self.dec.lm_head, self.cfg.vocab, self.top, self.logit_rows
        q, s, r = acts
        check(self.lib.rbn_matmul_t2_i8(self.ctx.handle, q.ptr + row0 * self.ctx.act_pitch(head.K), s.ptr + 4 * row0,
                                        r.ptr + 4 * row0, head.tiled.ptr, head.scale, M, head.K, V, None, self.logits.ptr))
        lp = self.stats.ptr
        check(self.lib.rbn_token_logprobs_f32(
            self.ctx.handle, self.logits.ptr, M, V, V, self.targets.ptr + 4 * row0 if with_targets else None, top,
            lp if with_targets else None, lp + 4 * R, lp + 8 * R, lp + 4 * R * (2 + top)))

    def _fetch(self, M: int):
        """(log probabilities of the targets, entropies, top tokens [M, top], their log probabilities)."""
        top, R = self.top, self.logit_rows
        raw = self.stats.download(np.uint32, R * (2 + 2 * top))
        tok = raw[2 * R:2 * R + M * top].view(np.int32).reshape(M, top)
        lps = raw[R * (2 + top):R * (2 + top) + M * top].view(np.float32).reshape(M, top)
        return raw[:M].view(np.float32).copy(), raw[R:R + M].view(np.float32).copy(), tok.copy(), lps.copy()

    # -- what the host knows before it queues anything --------------------------------------------------
    def _check_known(self):
        if self._lost:
            raise RuntimeError("an earlier call failed and what the device holds is unknown")

    def _check_room(self, new: dict) -> int:
        """Refuses `new` tokens per row that the device would refuse; returns how many pages they need."""
        self._check_known()
        total = sum(new.values())
        if total > self.max_tokens:
            raise ValueError("%d tokens in one call: max_tokens is %d" % (total, self.max_tokens))
        blocks = lambda n: -(-int(n) // _lib.KV_BLOCK)  # noqa: E731
        need = 0
        for r, n in new.items():
            if self._len[r] + n > self.cfg.max_seq:
                raise ValueError("row %d would hold %d positions: max_seq is %d" % (r, self._len[r] + n, self.cfg.max_seq))
            need += blocks(self._len[r] + n) - blocks(self._len[r])
        if need > self._free:
            raise ValueError("%d pages are needed, %d are free" % (need, self._free))
        return need

    @contextlib.contextmanager
    def _admitted(self, new: dict):
        """Books `new` tokens per row for the work queued inside.  Where that fails, the host's copies are brought in line with
        the device, and rows that had advanced there, whose new positions may hold nothing, end."""
        before, need = self._len.copy(), self._check_room(new)
        try:
            self._upload_counts(new)
            self._free -= need
            for r, n in new.items():
                self._len[r] += n
            yield sum(new.values())
        except BaseException:
            try:
                self._len = self.cache.lengths().astype(np.int64)
                self._free = self.cache.free_pages()
                ended = [r for r in new if self._len[r] != before[r]]
                if ended:
                    self._release(ended)
                for r in ended:
                    self._next.pop(r, None)
            except Exception:
                self._lost = True
            raise

    def _upload_counts(self, new: dict):
        counts = np.zeros(self.rows, dtype=np.int32)
        for r, n in new.items():
            counts[r] = n
        self.d_new.upload(counts)

    def _release(self, rows):
        self._upload_counts({r: -1 for r in rows})
        self.cache.plan(self.d_new)
        for r in rows:
            self._free += -(-int(self._len[r]) // _lib.KV_BLOCK)
            self._len[r] = 0

    def _prompts(self, prompts: dict) -> dict:
        out = {}
        for r, ids in sorted(prompts.items()):
            ids = np.asarray(ids)
            if not 0 <= r < self.rows:
                raise ValueError("row %d is outside [0, %d)" % (r, self.rows))
            if r in self._next:
                raise ValueError("row %d is running" % r)
            if ids.ndim != 1 or ids.size == 0:
                raise ValueError("a prompt must be a non-empty vector of token ids")
            if not (ids.min() >= 0 and ids.max() < self.cfg.vocab):
                raise ValueError("the prompt of row %d has token ids outside [0, %d)" % (r, self.cfg.vocab))
            out[r] = np.ascontiguousarray(ids, dtype=np.int32)
        if not out:
            raise ValueError("no prompts")
        return out

    # -- serving -------------------------------------------------------------------------------------
    @property
    def running(self) -> dict:
        """Running rows and the token each of them will take next."""
        return dict(self._next)

    def start(self, prompts: dict) -> dict:
        """Puts prompts (row -> token ids) into free rows; returns row -> NextToken."""
        prompts = self._prompts(prompts)
        ids = np.concatenate(list(prompts.values()))
        with self._admitted({r: p.size for r, p in prompts.items()}):
            self.tokens.upload(ids)
            self._forward(ids.size, max(p.size for p in prompts.values()))
            # the last token of each prompt
            pitch = self.ctx.act_pitch(self.cfg.hidden)
            ends = np.cumsum([p.size for p in prompts.values()]) - 1
            for i, e in enumerate(ends):
                for src, dst, n in zip(self.acts, self.last, (pitch, 4, 4)):
                    check(self.lib.rbn_d2d(self.ctx.handle, dst.ptr + i * n, src.ptr + int(e) * n, n))
            self._logprobs(self.last, 0, len(ends), False)
            got = self._fetch(len(ends))
        return self._took(list(prompts), *got[1:])

    def _took(self, rows, entropy, tok, lps) -> dict:
        got = {r: NextToken(int(tok[i, 0]), float(lps[i, 0]), float(entropy[i]), tok[i], lps[i]) for i, r in enumerate(rows)}
        self._next.update(got)
        return got

    def step(self, use_graph: bool = True) -> dict:
        """Appends its next token to every running row; returns row -> NextToken (the one after it).  The step of a
        number of running rows is captured once and replayed."""
        rows = sorted(self._next)
        if not rows:
            raise ValueError("no row is running")
        new, M = {r: 1 for r in rows}, len(rows)
        if use_graph and M not in self._graphs:
            self._check_room(new)
            self._graphs[M] = self._capture_step(M)
        with self._admitted(new):
            self.tokens.upload(np.array([self._next[r].token for r in rows], dtype=np.int32))
            if use_graph:
                self.ctx.graph_launch(self._graphs[M])
            else:
                self._queue_step(M)
            got = self._fetch(M)
        return self._took(rows, *got[1:])

    def _capture_step(self, M: int):
        self.ctx.graph_begin()
        try:
            self._queue_step(M)
        except BaseException:
            # the capture has to end; a graph of a part of the step is of no use
            with contextlib.suppress(_lib.RbnError):
                self.ctx.graph_destroy(self.ctx.graph_end())
            raise
        return self.ctx.graph_end()

    def _queue_step(self, M: int):
        self._forward(M, 1)
        self._logprobs(self.acts, 0, M, False)

    def finish(self, rows):
        """Ends rows; their pages are free again."""
        rows = [rows] if isinstance(rows, (int, np.integer)) else list(rows)
        if len(set(rows)) != len(rows) or any(r not in self._next for r in rows):
            raise ValueError("rows %s are not all running" % rows)
        self._check_known()
        self._release(rows)
        for r in rows:
            del self._next[r]

    def score(self, prompts: dict):
        """Log probabilities of given tokens: for each prompt (row -> token ids, free rows) the log probability of its
        tokens 1 .. and the entropy before each of them: row -> (logprobs [n-1], entropies [n-1]).  The rows are
        free again afterwards."""
        prompts = self._prompts(prompts)
        ids = np.concatenate(list(prompts.values()))
        # token i is followed by token i + 1 of its own prompt; the last one has no target
        targets = np.concatenate([np.append(p[1:], -1) for p in prompts.values()]).astype(np.int32)
        lp, ent = [], []
        with self._admitted({r: p.size for r, p in prompts.items()}):
            self.tokens.upload(ids)
            self.targets.upload(targets)
            self._forward(ids.size, max(p.size for p in prompts.values()))
            for at in range(0, ids.size, self.logit_rows):
                n = min(self.logit_rows, ids.size - at)
                self._logprobs(self.acts, at, n, True)
                got = self._fetch(n)
                lp.append(got[0])
                ent.append(got[1])
            self._release(list(prompts))
        lp, ent = np.concatenate(lp), np.concatenate(ent)
        out, at = {}, 0
        for r, p in prompts.items():
            out[r] = (lp[at:at + p.size - 1], ent[at:at + p.size - 1])
            at += p.size
        return out

    def close(self):
        """Destroys the captured steps."""
        for g in self._graphs.values():
            self.ctx.graph_destroy(g)
        self._graphs = {}
