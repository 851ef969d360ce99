"""CPU checks of the host side of the key/value cache ops where calls meet: threads, devices, sizes."""
import threading

import torch

from nemotron_ops_b200 import ops


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
