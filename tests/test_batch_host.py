"""The batched serving operators without a GPU: page layouts and indexing (kv_index.h compiled for the
host), refusals of bad arguments, size rules, and the numpy model the GPU tests compare with."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import batch_model as BM
from ronn_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("kv") / "kv_host.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover",
                    os.path.join(ROOT, "tests", "host", "kv_host.cpp"), "-o", out], check=True)
    return C.CDLL(out)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    return _lib.load()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("which", [0, 1])
def test_page_layout_is_a_permutation(host, hd, which):
    at = [host.kv_byte(which, hd, t, d) for t in range(32) for d in range(hd)]
    assert sorted(at) == list(range(32 * hd))
    # and the one that the header states
    for t in (0, 5, 16, 31):
        for d in (0, 7, 8, 33, hd - 1):
            k = ((t // 16 * (hd // 64) + d // 64) * 64 + d % 32 // 8 * 16 + t % 16) * 16 + d // 32 % 2 * 8 + d % 8
            v = (d // 32 * 64 + t % 16 // 4 * 16 + d % 16) * 16 + d // 16 % 2 * 8 + t // 16 * 4 + t % 4
            assert host.kv_byte(which, hd, t, d) == (v if which else k)


def units(host, rows, max_blocks, batch, u):
    arr = {k: np.asarray(batch[k], dtype=np.int32) for k in ("start", "row", "pos", "unit", "count")}
    arr["unit"] = np.concatenate([arr["unit"], np.full(len(arr["row"]) - len(arr["unit"]), -1, np.int32)])
    out = (C.c_int * 7)()
    p = lambda k: arr[k].ctypes.data_as(C.c_void_p)  # noqa: E731
    bad = host.kv_unit_of(rows, max_blocks, len(arr["row"]), p("start"), p("row"), p("pos"), p("unit"), p("count"), u, out)
    return bool(bad), list(out)


def test_units_of_a_planned_batch(host):
    rng = np.random.default_rng(3)
    rows, max_blocks, pages = 9, 16, 200
    length = rng.integers(0, 300, rows)
    new = rng.integers(0, 150, rows)
    new[2] = 0
    table = rng.permutation(pages)[:rows * max_blocks].reshape(rows, max_blocks).astype(np.int32)
    p = BM.plan(length, new, table, np.arange(pages, dtype=np.int32), (0, pages), 2000)
    batch = dict(p, count=[len(p["row"]), len(p["unit"])])
    seen = np.zeros(len(p["row"]), int)
    for u in range(len(p["unit"])):
        bad, (row, first, n, pos, row_first, row_pos, row_n) = units(host, rows, max_blocks, batch, u)
        assert not bad and n >= 1 and pos // 32 == (pos + n - 1) // 32
        assert (p["row"][first:first + n] == row).all() and (p["pos"][first:first + n] == pos + np.arange(n)).all()
        assert (row_first, row_pos, row_n) == (p["start"][row], length[row], new[row])
        seen[first:first + n] += 1
    assert (seen == 1).all()
    assert units(host, rows, max_blocks, batch, len(p["unit"]))[1][2] == 0


def test_bad_numbers_are_left_out(host):
    good = dict(start=[0, 3, 3], row=[0, 0, 0, -7], pos=[30, 31, 32, -7], unit=[0, 2, -7, -7], count=[3, 2])
    assert not units(host, 2, 4, good, 0)[0] and units(host, 2, 4, good, 0)[1][2] == 2
    for key, at, value in (("unit", 0, -1), ("unit", 0, 3), ("unit", 0, 1 << 30), ("row", 0, -1), ("row", 0, 2),
                           ("pos", 0, -5), ("pos", 0, 128), ("pos", 0, 2 ** 31 - 1), ("start", 0, 1), ("start", 0, -1),
                           ("start", 1, 0), ("start", 1, 4), ("start", 1, 1 << 30), ("pos", 0, 127)):
        b = {k: list(v) for k, v in good.items()}
        b[key][at] = value
        bad, out = units(host, 2, 4, b, 0)
        assert bad and out[2] == 0, (key, value)
    b = dict(good, count=[1 << 30, 1 << 30])        # more than the arrays hold: nothing behind them is read
    assert units(host, 2, 4, b, 4)[1][2] == 0
    b = dict(good, count=[-1, -1])
    assert units(host, 2, 4, b, 0)[1][2] == 0


def test_bad_pages_are_left_out(host):
    table = np.array([[0, 9, -1, 10], [2 ** 31 - 1, -2 ** 31, 3, 4]], dtype=np.int32)
    got = [[host.kv_page_of(2, 4, 10, table.ctypes.data_as(C.c_void_p), r, b) for b in range(4)] for r in range(2)]
    assert got == [[0, 9, -1, -1], [-1, -1, 3, 4]]
    assert [host.kv_slot_page_of(10, s) for s in (0, 31, 32, 319, 320, -1, -32, -33, 2 ** 31 - 1, -2 ** 31)] == \
        [0, 0, 1, 9, -1, -1, -1, -1, -1, -1]


def test_size_rules(lib):
    assert lib.rbn_kv_code_bytes(1000, 5, 128) == 1000 * 5 * 32 * 128
    assert lib.rbn_kv_scale_bytes(1000, 5) == 20000
    assert lib.rbn_kv_open_bytes(16, 20, 64) == 16 * 20 * 32 * 64 * 2
    assert lib.rbn_kv_code_bytes(60_000_000, 1024, 128) == 60_000_000 * 1024 * 32 * 128      # no 32-bit wrap
    for bad in ((1 << 26, 1, 128), (10, 1025, 128), (10, 1, 96)):
        assert lib.rbn_kv_code_bytes(*bad) == 0
    assert lib.rbn_kv_open_bytes(2049, 1, 128) == 0 and lib.rbn_kv_scale_bytes(1 << 26, 1) == 0


# Arguments are looked at before the context, so every refusal shows without a device: what is
# sound gets as far as "context is NULL".
def sound():
    p = 0x10000   # never dereferenced on the host
    return (_lib.KvTable(4, 8, 100, p, p, p, p), _lib.KvBatch(64, p, p, p, p, p, p),
            _lib.KvLayer(0, 4, 128, 0, p, p, p, p, p, p))


def calls(lib, t, b, l, heads=8, theta=1e4, new=0x20000, out=0x20000, state=0x20000, q=0x20000, qkv=0x20000, count=5,
          max_new=1):
    return {
        "plan": lambda: lib.rbn_kv_plan(None, t, new, b, out, state),
        "store": lambda: lib.rbn_rope_kv_store_q8(None, qkv, t, b, l, heads, theta, q),
        "read": lambda: lib.rbn_kv_read_f16(None, t, l, new, new, count, out, out),
        "attend": lambda: lib.rbn_attention_q8kv(None, q, t, b, l, heads, max_new, out),
    }


def message(lib, call):
    assert call() == _lib.RBN_ERR_INVALID
    return lib.rbn_last_error().decode()


def test_sound_arguments_reach_the_context(lib):
    for call in calls(lib, *sound()).values():
        assert message(lib, call) == "context is NULL"


@pytest.mark.parametrize("struct,field,value,names,word", [
    (0, "rows", 0, "plan store read attend", "bad sizes"), (0, "rows", 2049, "plan store read attend", "bad sizes"),
    (0, "max_blocks", 0, "plan store read attend", "bad sizes"),
    (0, "max_blocks", (1 << 20) + 1, "plan store read attend", "bad sizes"),
    (0, "pages", 0, "plan store read attend", "bad sizes"), (0, "pages", 1 << 26, "plan store read attend", "bad sizes"),
    (0, "rows", 1 << 63, "plan store read attend", "bad sizes"),
    (0, "d_table", None, "plan store read attend", "null pointer"), (0, "d_len", None, "plan store read attend", "null pointer"),
    (0, "d_ring", None, "plan", "null pointer"), (0, "d_ring_state", None, "plan", "null pointer"),
    (1, "max_tokens", 0, "plan store attend", "max_tokens"), (1, "max_tokens", (1 << 18) + 1, "plan store attend", "max_tokens"),
    (1, "d_start", None, "plan store attend", "null pointer"), (1, "d_row", None, "plan store attend", "null pointer"),
    (1, "d_pos", None, "plan store attend", "null pointer"), (1, "d_slot", None, "plan store attend", "null pointer"),
    (1, "d_unit", None, "plan store attend", "null pointer"), (1, "d_count", None, "plan store attend", "null pointer"),
    (2, "format", 2, "store read attend", "format"), (2, "kv_heads", 0, "store read attend", "kv_heads"),
    (2, "kv_heads", 1025, "store read attend", "kv_heads"), (2, "head_dim", 96, "store read attend", "head_dim 64 or 128"),
    (2, "head_dim", 0, "store read attend", "head_dim"), (2, "d_k", None, "store read attend", "null pointer"),
    (2, "d_v", None, "store read attend", "null pointer"), (2, "d_k_open", None, "store read attend", "null pointer"),
    (2, "d_v_open", None, "store read attend", "null pointer"), (2, "d_k_scale", None, "store read attend", "null pointer"),
    (2, "d_v_scale", None, "store read attend", "null pointer"), (2, "d_k", 0x10008, "store read attend", "aligned"),
    (2, "d_v", 0x10004, "store read attend", "aligned"), (2, "d_k_open", 0x10002, "store read attend", "aligned"),
    (2, "d_v_open", 0x10008, "store read attend", "aligned"),
])
def test_bad_descriptors_are_refused(lib, struct, field, value, names, word):
    args = sound()
    setattr(args[struct], field, value)
    for name in names.split():
        assert word in message(lib, calls(lib, *args)[name]), (name, field, value)


@pytest.mark.parametrize("kw,names,word", [
    (dict(new=None), "plan read", "null pointer"), (dict(out=None), "plan read attend", "null pointer"),
    (dict(state=None), "plan", "null pointer"), (dict(q=None), "store attend", "null pointer"),
    (dict(qkv=None), "store", "null pointer"), (dict(q=0x20004), "store attend", "aligned"),
    (dict(qkv=0x20008), "store", "aligned"), (dict(out=0x20008), "attend", "aligned"),
    (dict(heads=0), "store attend", "heads"), (dict(heads=9), "store attend", "multiple"),
    (dict(heads=1028), "store attend", "heads"), (dict(theta=0.0), "store", "theta"), (dict(theta=-1.0), "store", "theta"),
    (dict(theta=float("inf")), "store", "theta"), (dict(theta=float("nan")), "store", "theta"),
    (dict(count=0), "read", "count"), (dict(count=1 << 31), "read", "count"), (dict(max_new=0), "attend", "max_new"),
])
def test_bad_arguments_are_refused(lib, kw, names, word):
    for name in names.split():
        assert word in message(lib, calls(lib, *sound(), **kw)[name]), (name, kw)


def test_null_descriptors_are_refused(lib):
    t, b, l = sound()
    for args in ((None, b, l), (t, None, l), (t, b, None)):
        for name, call in calls(lib, *args).items():
            if (name == "plan" and args[2] is None) or (name == "read" and args[1] is None):
                continue
            assert "null pointer" in message(lib, call), name


def test_calls_of_too_many_workgroups_are_refused(lib):
    """A launch holds fewer than 2^32 threads: the largest calls within the ranges of the single arguments do not fit."""
    t, b, l = sound()
    assert "aligned" in message(lib, calls(lib, t, b, l, out=0x20008)["read"])
    b.max_tokens, l.kv_heads, t.rows = 1 << 18, 1024, 2048
    assert "too much" in message(lib, calls(lib, t, b, l, heads=1024)["attend"])
    assert "too much" in message(lib, calls(lib, t, b, l, heads=1024, max_new=2)["attend"])
    assert message(lib, calls(lib, t, b, l, heads=1024)["store"]) == "context is NULL"
    b.max_tokens = 1 << 13
    assert message(lib, calls(lib, t, b, l, heads=1024)["attend"]) == "context is NULL"
    assert message(lib, calls(lib, t, b, l, heads=1024, max_new=2)["attend"]) == "context is NULL"
    assert "too many places" in message(lib, calls(lib, t, b, l, count=(1 << 20) + 1)["read"])
    assert message(lib, calls(lib, t, b, l, count=(1 << 20) - 64)["read"]) == "context is NULL"


def test_logprobs_refusals(lib):
    p = 0x10000

    def call(logits=p, rows=3, vocab=100, pitch=100, target=p, top=2, lp=p, ent=p, tok=p, top_lp=p):
        return message(lib, lambda: lib.rbn_token_logprobs_f32(None, logits, rows, vocab, pitch, target, top, lp, ent, tok,
                                                               top_lp))
    assert call() == "context is NULL"
    assert call(target=None, lp=None) == "context is NULL" and call(ent=None) == "context is NULL"
    assert call(top=0, tok=None, top_lp=None) == "context is NULL"
    for kw, word in ((dict(logits=None), "null pointer"), (dict(rows=0), "bad sizes"), (dict(rows=1 << 20), "bad sizes"),
                     (dict(vocab=0), "bad sizes"), (dict(vocab=1 << 30, pitch=1 << 30), "bad sizes"),
                     (dict(pitch=99), "bad sizes"), (dict(top=33), "at most 32"), (dict(target=None), "go together"),
                     (dict(lp=None), "go together"), (dict(tok=None), "top needs"), (dict(top_lp=None), "top needs")):
        assert word in call(**kw), kw


def test_stream_context_needs_a_device(lib):
    if lib.rbn_device_count():
        pytest.skip("a GPU is visible")
    out = C.c_void_p()
    assert lib.rbn_ctx_create_on_stream(0, None, C.byref(out)) == _lib.RBN_ERR_NO_DEVICE and not out.value


def test_model_rounds_to_e4m3():
    """The model's e4m3 rounding against the table of the format's values: every midpoint goes to the even code."""
    v = np.array(sorted({abs(x) for x in BM.e4m3_values() if x == x}))
    assert v[-1] == 448.0 and v[1] == 2.0 ** -9 and len(v) == 127
    assert (BM.round_e4m3(v) == v).all()
    mid = (v[1:] + v[:-1]) / 2
    want = np.where(np.arange(126) % 2 == 0, v[:-1], v[1:])
    assert (BM.round_e4m3(mid) == want).all() and (BM.round_e4m3(-mid) == -want).all()
    assert (BM.round_e4m3(mid * (1 + 1e-9)) == v[1:]).all() and (BM.round_e4m3(mid * (1 - 1e-9)) == v[:-1]).all()


def test_c_structs_match_the_header():
    header = open(os.path.join(ROOT, "include", "ronn_bitnet_hip.h")).read()
    import re
    for name, struct in (("rbn_kv_table", _lib.KvTable), ("rbn_kv_batch", _lib.KvBatch), ("rbn_kv_layer", _lib.KvLayer)):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\}" % name, header, re.S).group(1), flags=re.S)
        fields = [f for decl in body.split(";") for f in re.findall(r"\*?(\w+)\s*(?:,|$)", decl.strip())]
        assert fields == [f for f, _ in struct._fields_]
        rust = open(os.path.join(ROOT, "rust", "ronn-bitnet-hip-sys", "src", "lib.rs")).read()
        m = re.search(r"pub struct %s \{(.*?)\}" % name, rust, re.S).group(1)
        assert fields == re.findall(r"pub (\w+):", m)
    for macro in ("RBN_KV_BLOCK", "RBN_KV_MAX_ROWS", "RBN_TOP_MAX", "RBN_FLAG_KV_REFUSED", "RBN_FLAG_KV_BAD_INDEX",
                  "RBN_FLAG_KV_NONFINITE"):
        value = re.search(r"#define %s (\d+)" % macro, header).group(1)
        assert int(value) == getattr(_lib, macro[4:])
        assert re.search(r"pub const %s: u\d+ = %s;" % (macro, value), rust), macro
