"""CPU checks of the key/value cache entry points: the C ABI refuses bad arguments before any device work, the
64-bit oracle agrees with the definitions on hand-made cases, and the Python ops take no CPU tensors."""
import ctypes

import numpy as np
import pytest
import torch

import oracle as O
from nemotron_ops_b200 import _lib, ops

NULL = ctypes.c_void_p(0)
SOME = ctypes.c_void_p(4096)  # aligned; never dereferenced on the host


def _sh(*dims):
    return _lib.shape_arg(dims)[0]


GOOD = dict(cache=(5, 2, 16, 128), table=(3, 4), rows=(3, 2, 4, 128), strides=(1024, 512), fmt=0, window=0, sinks=0)


def _attention(ptr=SOME, ws=1 << 40, **kw):
    a = dict(GOOD, **kw)
    lib = _lib.lib()
    rc = lib.bolt_kv_attention(ptr, _sh(*a["rows"]), _sh(*a["strides"]), ptr, _sh(*a["cache"]), ptr, ptr, ptr, ptr,
                               _sh(*a["table"]), ptr, ptr, 0.1, a["window"], a["sinks"], a["fmt"], ptr, ptr, ptr, ws,
                               NULL)
    return rc, _lib.last_error()


@pytest.mark.parametrize("kw,msg", [
    (dict(cache=(5, 2, 16, 96)), "KvAttention: head size must be 64 or 128"),
    (dict(cache=(5, 2, 24, 128)), "KvAttention: a page must hold 16, 32, 64, 128 or 256 tokens"),
    (dict(cache=(5, 2, 512, 128)), "KvAttention: a page must hold 16, 32, 64, 128 or 256 tokens"),
    (dict(cache=(0, 2, 16, 128)), "KvAttention: cache must be [pages, heads, tokens, head size]"),
    (dict(cache=(5, 0, 16, 128)), "KvAttention: cache must be [pages, heads, tokens, head size]"),
    (dict(cache=(1 << 26, 4, 16, 128)), "KvAttention: cache must have fewer than 2^31 rows"),
    (dict(table=(3, 1 << 27)), "KvAttention: page table must be"),
    (dict(table=(2, 4)), "KvAttention: rows must be [sequences, rows, heads, head size]"),
    (dict(rows=(3, 2, 3, 128)), "KvAttention: query heads must be a multiple of the cache's heads"),
    (dict(rows=(3, 2, 4, 64)), "KvAttention: rows must be [sequences, rows, heads, head size]"),
    (dict(rows=(3, -1, 4, 128)), "KvAttention: bad row count"),
    (dict(strides=(1024, 516)), "KvAttention: row strides must be multiples of 8"),
    (dict(strides=(-8, 512)), "KvAttention: row strides must be multiples of 8"),
    (dict(fmt=2), "KvAttention: unknown cache format"),
    (dict(window=-1), "KvAttention: window and sinks must not be negative"),
    (dict(sinks=-1), "KvAttention: window and sinks must not be negative"),
    (dict(ptr=NULL), "KvAttention: null buffer"),
    (dict(ptr=ctypes.c_void_p(4104)), "KvAttention: tensors must be 16-byte aligned"),
    (dict(ws=1000), "KvAttention: the workspace is too small"),
])
def test_attention_refusals(kw, msg):
    rc, err = _attention(**kw)
    assert rc == 1 and msg in err, err


def test_nothing_to_do_needs_no_buffers():
    for kw in (dict(rows=(3, 0, 4, 128)), dict(rows=(0, 2, 4, 128), table=(0, 4))):
        rc, err = _attention(ptr=NULL, ws=0, **kw)
        assert rc == 0 and err == ""


def test_workspace_size():
    lib = _lib.lib()
    # it grows with the rows a head of the cache serves, and not with sequences or lengths
    one = lib.bolt_kv_attention_workspace(_sh(3, 1, 4, 128), _sh(5, 2, 16, 128))
    many = lib.bolt_kv_attention_workspace(_sh(3, 500, 4, 128), _sh(5, 2, 16, 128))
    assert 0 < one < many < 1 << 26
    assert lib.bolt_kv_attention_workspace(_sh(3, 1, 3, 128), _sh(5, 2, 16, 128)) == -1
    assert "multiple" in _lib.last_error()


def test_other_refusals():
    lib = _lib.lib()
    c, t, r, s = _sh(5, 2, 16, 128), _sh(3, 4), _sh(3, 2, 2, 128), _sh(1024, 512)
    bad = _sh(1024, 500)
    assert lib.bolt_kv_append(SOME, r, s, SOME, bad, SOME, c, SOME, SOME, SOME, SOME, t, SOME, SOME, 0, NULL) == 1
    assert "KvAppend: row strides" in _lib.last_error()
    assert lib.bolt_kv_append(SOME, _sh(3, 2, 4, 128), s, SOME, s, SOME, c, SOME, SOME, SOME, SOME, t, SOME, SOME, 0,
                              NULL) == 1
    assert "KvAppend: rows must be" in _lib.last_error()
    assert lib.bolt_kv_read(SOME, c, SOME, SOME, SOME, SOME, t, SOME, SOME, -1, 0, SOME, SOME, NULL) == 1
    assert "KvRead: bad row count" in _lib.last_error()
    q = _sh(3, 2, 4, 128)
    assert lib.bolt_kv_score(SOME, q, s, SOME, c, SOME, SOME, t, SOME, SOME, SOME, 0.1, 0, 0, 0, SOME, 63, NULL) == 1
    assert "KvScore: score must cover the page table" in _lib.last_error()
    for keep, sinks, recent, width, sw, msg in [(0, 0, 0, 1, 64, "at least 1"), (8, 5, 4, 1, 64, "must not exceed keep"),
                                                (17, 0, 0, 1, 64, "must hold keep positions"),
                                                (8, 0, 0, 1, 63, "score must cover"), (8, -1, 0, 1, 64, "must not exceed")]:
        assert lib.bolt_kv_evict(SOME, c, SOME, SOME, SOME, SOME, t, SOME, SOME, sw, SOME, width, keep, sinks, recent,
                                 0, SOME, SOME, SOME, NULL) == 1
        assert msg in _lib.last_error()


def test_ops_take_no_cpu_tensors():
    u8 = torch.zeros(1, 1, 16, 64, dtype=torch.uint8)
    f, i = torch.zeros(1, 1), torch.zeros(1, 1, dtype=torch.int32)
    q = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    for call in (lambda: ops.KvAttention(q, u8, u8, f, f, i, i[0], i[0], 0.1),
                 lambda: ops.KvAppend(q, q, u8, u8, f, f, i, i[0], i[0]),
                 lambda: ops.KvRead(u8, u8, f, f, i, i[0], i[0], 1),
                 lambda: ops.KvAttention(q, None, u8, f, f, i, i[0], i[0], 0.1)):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            call()


# ---------------------------------------------------------------------------------------------
# the oracle on cases that can be written down
# ---------------------------------------------------------------------------------------------
def test_oracle_codes():
    assert O.kv_values(torch.tensor([1, 128, 255], dtype=torch.uint8), 0).tolist() == [-127.0, 0.0, 127.0]
    assert O.kv_values(torch.tensor([0x7E, 0xFE, 0x01, 0x38], dtype=torch.uint8), 1).tolist() == [448.0, -448.0, 2.0 ** -9, 1.0]


def test_oracle_mask():
    assert O.kv_visible(5, 9, 0, 0).tolist() == [True] * 6 + [False] * 3
    assert O.kv_visible(5, 9, 2, 1).tolist() == [True, False, False, False, True, True, False, False, False]


def test_oracle_attention_of_equal_keys_is_the_mean():
    k = torch.full((1, 1, 16, 64), 130, dtype=torch.uint8)
    v = torch.arange(16, dtype=torch.uint8).view(1, 1, 16, 1).expand(1, 1, 16, 64) + 128
    one = torch.ones(1, 1)
    q = torch.ones(1, 1, 2, 64).bfloat16()
    r = O.kv_attention(q, k, v.contiguous(), one, one, torch.zeros(1, 1, dtype=torch.int32), torch.tensor([6]),
                       torch.tensor([7]), 0.01)
    assert np.allclose(r["o"], 3.0) and np.allclose(r["lse"], 64 * 2 * 0.01 + np.log(7))
    s, added = O.kv_score(q, k, one, torch.zeros(1, 1, dtype=torch.int32), torch.tensor([6]), torch.tensor([7]),
                          torch.from_numpy(r["lse"]), torch.zeros(1, 1, 16), 0.01)
    assert np.allclose(added[0, 0, :7], 2 / 7) and not added[0, 0, 7:].any()


def test_oracle_eviction_order():
    keep = O.kv_evict_keep(np.array([5, 1, 3, 3, 3, 0, 9.0, 2]), 8, 5, 1, 1)
    assert keep.tolist() == [0, 2, 3, 6, 7]  # of the equal ones the lower
    assert O.kv_evict_keep(np.array([1.0, np.nan, 7, 2]), 4, 2, 0, 0).tolist() == [1, 2]
    assert O.kv_evict_keep(np.array([1.0, 2]), 2, 3, 0, 0).tolist() == [0, 1]
