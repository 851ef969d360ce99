"""CPU checks of the host side of the key/value cache ops where calls meet: threads, devices, sizes."""
import ctypes
import threading

import torch

from nemotron_ops_b200 import _lib, ops


def test_host_threads_do_not_share_scratch_memory(monkeypatch):
    # an attention call enqueues two kernels that meet in its scratch memory; another thread's call on the same
    # stream may be enqueued between them
    monkeypatch.setattr(ops, "_stream", lambda t: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    like = torch.zeros(1, dtype=torch.uint8)
    got, turn = [], threading.Barrier(3, timeout=60)

    def call(n):
        ws = ops._kv_workspace(like, n)
        turn.wait()  # all hold theirs at once
        got.append(ws)

    threads = [threading.Thread(target=call, args=(n,)) for n in (64, 64)]
    for t in threads:
        t.start()
    call(32)
    for t in threads:
        t.join()
    spans = sorted((w.data_ptr(), w.data_ptr() + w.numel()) for w in got)
    assert len(spans) == 3 and all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
    # calls of one thread and one stream follow one another and have one buffer, which grows
    one = ops._kv_workspace(like, 100)
    assert one.numel() == 100 and ops._kv_workspace(like, 10) is one


def test_more_rows_than_32_bits_count():
    # rows x query heads of a cache head: the kernels count them in 32 bits
    def sh(*dims):
        return _lib.shape_arg(dims)[0]

    lib, some = _lib.lib(), ctypes.c_void_p(4096)  # aligned; never dereferenced on the host
    cache, table, strides = sh(5, 2, 16, 128), sh(3, 4), sh(1024, 0)
    for rows, heads in ((1 << 29, 8), (1 << 29, 16), (65536, 2 << 15), (1 << 20, 2 << 12)):
        q = sh(3, rows, heads, 128)
        assert lib.bolt_kv_score(some, q, strides, some, cache, some, some, table, some, some, some, 0.1, 0, 0, 0, some,
                                 64, None) == 1
        assert "KvScore: rows times query heads of a cache head must be fewer than 2^31" in _lib.last_error()
        assert lib.bolt_kv_attention(some, q, strides, some, cache, some, some, some, some, table, some, some, 0.1, 0, 0,
                                     0, some, some, some, 1 << 40, None) == 1
        assert "KvAttention: rows times query heads of a cache head must be fewer than 2^31" in _lib.last_error()
