"""The paged 8-bit key/value cache ops where calls, values, pages and sizes are out of the ordinary.

Bounds are those of test_gpu_kv.py's head with one more term for o, which its formula leaves out: a weight (times
its page's V scale) below 2^-22 of the row's largest has fewer than 11 bits and errs by at most 2^-33 of that
largest, times the position's code.  It shows only where V scales are far apart; here they are within a factor of 6,
and it stays below the term of 2^-18 for the numbers of positions of these cases.
"""
import threading

import torch
import pytest

import test_gpu_kv as kv
from nemotron_ops_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


# ---------------------------------------------------------------------------------------------
# calls
# ---------------------------------------------------------------------------------------------
def test_host_threads_on_one_stream():
    # three threads enqueue attention calls of different shapes on the default stream: each as if it were alone
    shapes = [(4, 2, 16, 2, 128, 32, 0, [3000, 900, 0, 50]), (1, 1, 8, 1, 64, 16, 1, [20000]),
              (2, 40, 8, 2, 128, 16, 0, [700, 2100])]
    calls, want = [], []
    for i, (S, R, Hq, Hkv, D, T, fmt, lens) in enumerate(shapes):
        q, caches, scales, table, n = kv._large(S, R, Hq, Hkv, D, T, fmt, lens, seed=240 + i)
        calls.append(((q, *caches, *scales, table, (n - R).clamp(min=0), n, 0.1), dict(fmt=fmt)))
        want.append(ops.KvAttention(*calls[i][0], **calls[i][1]))
    torch.cuda.synchronize()
    got, turn = [[] for _ in shapes], threading.Barrier(len(shapes), timeout=60)

    def work(i):
        turn.wait()
        for _ in range(200):
            got[i].append(ops.KvAttention(*calls[i][0], **calls[i][1]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(shapes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for (o, lse), results in zip(want, got):
        assert len(results) == 200
        assert all(torch.equal(o, a) and torch.equal(lse, b) for a, b in results)
    assert ops.device_status() == 0
