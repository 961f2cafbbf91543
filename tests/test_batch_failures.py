"""BatchDecoder's own bookkeeping where a call fails on the way, without a GPU: buffers in host memory, the library's calls stubs that
do nothing, but for the page plan, which tests/batch_model.py does.  After a failure the host's lengths and free pages are the
device's, nothing is lost, and the decoder goes on."""
import os

import numpy as np
import pytest

import batch_model as BM
from ronn_amd import _lib
from ronn_amd.decoder import BatchDecoder, DecoderConfig


class Buffer:
    def __init__(self, owner, nbytes):
        self.owner, self.nbytes, self.data = owner, int(nbytes), np.zeros(int(nbytes), np.uint8)
        self.ptr = owner.next_ptr
        owner.next_ptr += (self.nbytes + 255) // 256 * 256 + 256
        owner.buffers[self.ptr] = self

    def upload(self, array):
        self.owner.call("upload")
        raw = np.ascontiguousarray(array).view(np.uint8).ravel()
        self.data[:raw.size] = raw
        return self

    def download(self, dtype, count, offset_bytes=0):
        self.owner.call("download")
        return self.data.view(np.uint8)[offset_bytes:offset_bytes + int(count) * np.dtype(dtype).itemsize].view(dtype).copy()

    def free(self):
        pass


class Device:
    """Context and library in one.  fail {name: n}: of the calls of that name, the one behind the next n raises; gone: all do."""

    def __init__(self):
        self.handle, self.lib, self.device = 1, self, 0
        self.next_ptr, self.buffers = 1 << 20, {}
        self.fail, self.gone, self.queue, self.graphs, self.live = {}, False, None, {}, 0
        self.real = _lib.load()

    def call(self, name):
        if name in self.fail:
            self.fail[name] -= 1
            if self.fail[name] < 0:
                if not self.gone:
                    del self.fail[name]
                raise _lib.RbnError(_lib.RBN_ERR_HIP, name + " fails")

    # the library
    def __getattr__(self, name):
        if not name.startswith("rbn_"):
            raise AttributeError(name)
        if name.endswith("_bytes"):
            return getattr(self.real, name)

        def stub(*args):
            self.call(name)
            if name == "rbn_kv_plan":
                if self.queue is not None:
                    self.queue.append(args)
                else:
                    self.plan(*args)
            return _lib.RBN_OK
        return stub

    def plan(self, handle, t, d_new, b, d_len_out, d_state_out):
        i32 = lambda p, n: self.buffers[p].data.view(np.int32)[:n]  # noqa: E731
        table, ring = i32(t.d_table, t.rows * t.max_blocks).reshape(t.rows, -1), i32(t.d_ring, t.pages)
        length, state = i32(t.d_len, t.rows), i32(t.d_ring_state, 2)
        p = BM.plan(length, i32(d_new, t.rows), table, ring, state, b.max_tokens)
        assert p["flags"] == 0
        table[:], ring[:], length[:], state[:] = p["table"], p["ring"], p["len_out"], p["ring_state_out"]

    # the context
    def alloc(self, nbytes):
        return Buffer(self, nbytes)

    def to_device(self, array):
        a = np.ascontiguousarray(array)
        return self.alloc(max(a.nbytes, 1)).upload(a)

    def act_pitch(self, k):
        return (k + 127) // 128 * 128

    def matmul(self, *args, **kw):
        self.call("matmul")

    def graph_begin(self):
        self.call("graph_begin")
        assert self.queue is None
        self.queue = []

    def graph_end(self):
        q, self.queue = self.queue, None       # the capture ends in any case
        self.call("graph_end")
        self.live += 1
        g = len(self.graphs) + 1
        self.graphs[g] = q
        return g

    def graph_launch(self, g):
        self.call("graph_launch")
        for args in self.graphs[g]:
            self.plan(*args)

    def graph_destroy(self, g):
        self.live -= 1


class Weights:
    """What BatchDecoder needs of a BitNetDecoder."""

    def __init__(self, dev, cfg):
        lin = type("Linear", (), dict(tiled=dev.alloc(1), scale=1.0, K=cfg.hidden, N=cfg.hidden))()
        vec = dev.alloc(1)
        self.ctx, self.cfg, self.embed, self.g_final, self.lm_head = dev, cfg, vec, vec, lin
        self.blocks = [dict(g_attn=vec, g_attn_sub=vec, g_ffn=vec, g_ffn_sub=vec, wqkv=lin, wo=lin, wgu=lin, wdown=lin)] * 2


PAGES = 12


@pytest.fixture
def decoder():
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    dev = Device()
    cfg = DecoderConfig(layers=2, hidden=256, heads=2, head_dim=128, ffn=384, vocab=100, max_seq=128)
    return BatchDecoder(Weights(dev, cfg), rows=4, pages=PAGES, max_tokens=200), dev


def consistent(dec, running):
    """Host and device agree, and the pages are the running rows' or free."""
    held = {r: n for r, n in enumerate(dec.cache.lengths()) if n}
    assert held == running and sorted(dec.running) == sorted(running)
    assert dec.cache.free_pages() == PAGES - sum(BM.blocks(n) for n in running.values()) == dec._free
    assert list(dec._len) == [running.get(r, 0) for r in range(dec.rows)]


# where a start or a score can fail: name and how many calls of it pass first (what runs before the plan and behind it)
PLACES = [("upload", 0), ("upload", 1), ("rbn_kv_plan", 0), ("rbn_embed_f32", 0), ("matmul", 0), ("rbn_attention_q8kv", 0), ("rbn_attention_q8kv", 1),
          ("rbn_token_logprobs_f32", 0), ("download", 0)]


@pytest.mark.parametrize("name,passing", PLACES + [("rbn_d2d", 4)])
def test_a_failed_start(decoder, name, passing):
    dec, dev = decoder
    dec.start({3: [1] * 33})
    dev.fail = {name: passing}
    with pytest.raises(_lib.RbnError, match=name):
        dec.start({0: [1] * 50, 2: [2] * 7})
    consistent(dec, {3: 33})
    dec.start({0: [1] * 100, 2: [2] * 90})
    consistent(dec, {0: 100, 2: 90, 3: 33})


@pytest.mark.parametrize("name,passing", PLACES + [("upload", 2), ("upload", 3), ("rbn_kv_plan", 1)])
def test_a_failed_score(decoder, name, passing):
    dec, dev = decoder
    dec.start({1: [1] * 64})
    dev.fail = {name: passing}
    with pytest.raises(_lib.RbnError, match=name):
        dec.score({0: [1] * 50, 2: [2] * 7})
    consistent(dec, {1: 64})
    dec.score({0: [1] * 100, 2: [2] * 90})
    consistent(dec, {1: 64})


@pytest.mark.parametrize("name,passing", PLACES)
def test_a_failed_eager_step(decoder, name, passing):
    """A step that the device has not begun leaves its rows as they were; one that it has ends them."""
    dec, dev = decoder
    dec.start({0: [1] * 63, 2: [2] * 7})
    dec.step(use_graph=False)
    dev.fail = {name: passing}
    with pytest.raises(_lib.RbnError, match=name):
        dec.step(use_graph=False)
    left = {0: 64, 2: 8} if name in ("upload", "rbn_kv_plan") else {}
    consistent(dec, left)
    if not left:
        dec.start({0: [1] * 64, 2: [2] * 8})
    dec.step(use_graph=False)
    consistent(dec, {0: 65, 2: 9})


@pytest.mark.parametrize("name,passing", [("graph_begin", 0), ("matmul", 0), ("rbn_kv_plan", 0), ("rbn_attention_q8kv", 1),
                                          ("rbn_token_logprobs_f32", 0), ("graph_end", 0), ("upload", 0), ("upload", 1),
                                          ("graph_launch", 0), ("download", 0)])
def test_a_failed_graph_step(decoder, name, passing):
    """A failed capture ends, leaves no graph and no changes; the next step captures anew."""
    dec, dev = decoder
    dec.start({0: [1] * 63, 2: [2] * 7})
    dev.fail = {name: passing}
    with pytest.raises(_lib.RbnError, match=name):
        dec.step()
    assert dev.queue is None
    left = {0: 63, 2: 7} if name != "download" else {}
    consistent(dec, left)
    if not left:
        dec.start({0: [1] * 63, 2: [2] * 7})
    dec.step()
    dec.step()
    consistent(dec, {0: 65, 2: 9})
    assert dev.live == 1 == len(dec._graphs)
    dec.close()
    assert dev.live == 0


def test_a_capture_that_neither_goes_on_nor_ends(decoder):
    dec, dev = decoder
    dec.start({0: [1] * 5})
    dev.fail = {"matmul": 2, "graph_end": 0}
    with pytest.raises(_lib.RbnError, match="matmul"):      # what went wrong first
        dec.step()
    consistent(dec, {0: 5})
    dec.step()
    consistent(dec, {0: 6})


@pytest.mark.parametrize("name", ["upload", "rbn_kv_plan"])
def test_a_failed_finish(decoder, name):
    dec, dev = decoder
    dec.start({0: [1] * 63, 2: [2] * 7})
    dev.fail = {name: 0}
    with pytest.raises(_lib.RbnError, match=name):
        dec.finish([0, 2])
    consistent(dec, {0: 63, 2: 7})
    dec.finish([0, 2])
    consistent(dec, {})


def test_refusals_come_before_anything_is_queued(decoder):
    dec, dev = decoder
    dec.start({0: [1] * 128, 1: [1] * 64})
    dev.fail = {name: 0 for name in ("upload", "graph_begin", "rbn_kv_plan", "download")}
    for call in (dec.step, lambda: dec.step(use_graph=False), lambda: dec.start({2: [1] * 129}), lambda: dec.start({2: [1] * 128, 3: [1] * 128}),
                 lambda: dec.score({2: [1] * 100, 3: [1] * 101})):
        with pytest.raises(ValueError):
            call()
    dev.fail = {}
    consistent(dec, {0: 128, 1: 64})


def test_token_ids_outside_the_vocabulary_are_refused(decoder):
    """(On the device an id would be clamped and, as a token to be scored, have a log probability of 0.)"""
    dec, dev = decoder
    dev.fail = {name: 0 for name in ("upload", "rbn_kv_plan", "download")}
    for ids in ([5, 100], [-1], [3, 2 ** 31 + 5], np.array([1, 2 ** 32], np.int64), np.array([2 ** 63 + 1], np.uint64), [1.0, float("nan")]):
        for call in (dec.start, dec.score):
            with pytest.raises(ValueError, match="outside"):
                call({0: [1, 2], 1: ids})
    dev.fail = {}
    consistent(dec, {})
    dec.score({0: [0, 99], 1: [99]})


def test_a_device_that_is_gone(decoder):
    """Where not even the lengths can be read back, nothing that follows is done on a guess."""
    dec, dev = decoder
    dec.start({0: [1] * 5})
    dev.fail, dev.gone = {"rbn_embed_f32": 0, "download": 0}, True
    with pytest.raises(_lib.RbnError, match="embed"):
        dec.step(use_graph=False)
    dev.fail = {}
    for call in (dec.step, lambda: dec.start({1: [1]}), lambda: dec.score({1: [1]}), lambda: dec.finish(0)):
        with pytest.raises(RuntimeError, match="unknown"):
            call()
