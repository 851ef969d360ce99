"""CPU checks of the host side of the key/value cache ops where calls meet: threads, devices, sizes."""
import ctypes
import threading

import pytest
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


class _On(torch.Tensor):
    """A host tensor that says it is on CUDA device `index`."""

    index = 0
    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", self.index))

    def get_device(self):
        return self.index


def _on(index, *shape, dtype=torch.float32):
    t = torch.zeros(*shape, dtype=dtype).as_subclass(_On)
    t.index = index
    return t


def _calls(where):
    """name -> (op, its tensors), each tensor on the device that where(op, argument) gives."""
    def make(op, **kinds):
        u8, f32, i32, bf16 = torch.uint8, torch.float32, torch.int32, torch.bfloat16
        forms = dict(k_cache=((5, 2, 16, 64), u8), v_cache=((5, 2, 16, 64), u8), k_scale=((5, 2), f32),
                     v_scale=((5, 2), f32), table=((3, 4), i32), start=((3,), i32), lens=((3,), i32),
                     q=((3, 2, 4, 64), bf16), k=((3, 2, 2, 64), bf16), v=((3, 2, 2, 64), bf16), lse=((3, 2, 4), f32),
                     score=((3, 2, 64), f32), new_table=((3, 1), i32))
        return {a: _on(where(op, a), *forms[a][0], dtype=forms[a][1]) for a in kinds["args"].split()}

    cache = "k_cache v_cache k_scale v_scale table lens"
    return [(ops.KvAppend, make("KvAppend", args=cache + " start k v"), {}),
            (ops.KvRead, make("KvRead", args=cache + " start"), dict(rows=2)),
            (ops.KvAttention, make("KvAttention", args=cache + " start q"), dict(scale=0.1)),
            (ops.KvScore, make("KvScore", args="k_cache k_scale table lens start q lse score"), dict(scale=0.1)),
            (ops.KvEvict, make("KvEvict", args=cache + " score new_table"), dict(keep=8))]


def test_tensors_of_two_devices(monkeypatch):
    # a kernel would take the other device's address for its own
    class Reached(Exception):
        pass

    def reached():
        raise Reached

    monkeypatch.setattr(ops, "lib", reached)  # nothing is launched
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(ops, "_stream", lambda t: 0)
    for op, tensors, rest in _calls(lambda op, arg: 0):
        with pytest.raises(Reached):
            op(**tensors, **rest)
        for other in tensors:
            mixed = dict(next(c for c in _calls(lambda o, arg: int(arg == other)) if c[0] is op)[1])
            with pytest.raises(RuntimeError, match=f"{op.__name__}: tensors must be on the current device"):
                op(**mixed, **rest)
    for op, tensors, rest in _calls(lambda op, arg: 1):  # all on one, which is not the current one
        with pytest.raises(RuntimeError, match=f"{op.__name__}: tensors must be on the current device"):
            op(**tensors, **rest)
