"""DecoderConfig: K/V heads that were not given follow the query heads, also in copies and after a change."""
import copy
import dataclasses
import pickle

import pytest

from ronn_amd.decoder import DecoderConfig


def test_kv_heads_follow_the_heads_unless_given():
    cfg = DecoderConfig()
    assert cfg.kv_heads == 20 and cfg.qkv_dim == 3 * cfg.attn_dim
    for other in (dataclasses.replace(cfg, heads=8), DecoderConfig(**{**dataclasses.asdict(cfg), "heads": 8}),
                  dataclasses.replace(dataclasses.replace(cfg, layers=2), heads=8)):
        assert other.kv_heads == 8 and other.qkv_dim == 3 * 8 * 128
    for same in (copy.copy(cfg), copy.deepcopy(cfg), pickle.loads(pickle.dumps(cfg))):
        assert same == cfg and repr(same) == repr(cfg)
        same.heads = 6
        assert same.kv_heads == 6 and same.qkv_dim == 3 * same.attn_dim
    assert cfg.kv_heads == 20


def test_given_kv_heads_stay():
    cfg = DecoderConfig(heads=20, kv_heads=5)
    assert dataclasses.replace(cfg, heads=10).kv_heads == 5 and dataclasses.replace(cfg, layers=1).qkv_dim == 30 * 128
    cfg.heads = 40
    assert cfg.kv_heads == 5
    cfg.kv_heads = 0
    assert cfg.kv_heads == 40
    equal = DecoderConfig(heads=4, kv_heads=4)           # given, though they are as many
    assert equal == DecoderConfig(heads=4)
    for bad in (dict(heads=6, kv_heads=4), dict(heads=6, kv_heads=-6), dict(heads=6, kv_heads=12)):
        with pytest.raises(ValueError, match="multiple"):
            DecoderConfig(**bad)
    with pytest.raises(ValueError, match="multiple"):
        dataclasses.replace(cfg, heads=6, kv_heads=5)
