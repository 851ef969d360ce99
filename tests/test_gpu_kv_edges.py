"""The paged 8-bit key/value cache ops where calls, values, pages and sizes are out of the ordinary.

Bounds are those of test_gpu_kv.py's head with one more term for o, which its formula leaves out: a weight (times
its page's V scale) below 2^-22 of the row's largest has fewer than 11 bits and errs by at most 2^-33 of that
largest, times the position's code.  It shows only where V scales are far apart; here they are within a factor of 6,
and it stays below the term of 2^-18 for the numbers of positions of these cases.
"""
import threading

import numpy as np
import pytest
import torch

import oracle as O
import test_gpu_kv as kv
from nemotron_ops_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"

ROWS = [(1, 1), (1, 8), (2, 8), (1, 17), (3, 8), (65, 2)]  # R, G: tiles of 8, of 16, and the tensor-memory kernel


def _check(o, lse, ref, D, bad):
    """The rows of `bad` [S, R, Hq] are NaN throughout, the others right."""
    o, lse = o.cpu().clone(), lse.cpu().clone()
    bad = torch.from_numpy(bad)
    assert bool(o[bad].isnan().all()) and bool(lse[bad].isnan().all())
    o[bad] = torch.from_numpy(ref["o"])[bad].to(o.dtype)
    lse[bad] = torch.from_numpy(ref["lse"])[bad].to(lse.dtype)
    kv._check_attention(o, lse, ref, D)


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


# ---------------------------------------------------------------------------------------------
# values that are not finite
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("value", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("R,G", ROWS)
def test_a_query_row_that_is_not_finite(R, G, D, fmt, value):
    # its o and lse are NaN, its neighbours' are as they were; rows that do not exist stay empty
    lens = [1500, 0, 90]
    c = kv.Cache(lens, 2, D, 16, fmt, seed=201)
    q = kv._rows(3, R, 2 * G, D, seed=202)
    start = (c.lens - R).clamp(min=0)
    if R > 1:
        start[2] = c.lens[2] - 1  # one row of R
    ref = O.kv_attention(q, *c.host(), c.table, start, c.lens, D ** -0.5, fmt=fmt)
    dirty, bad = q.clone(), np.zeros(q.shape[:3], dtype=bool)
    for s, r, i, d in ((0, R // 2, G, D - 1), (1, 0, 0, 3), (2, 0, G - 1, 0), (2, R - 1, G, 5)):
        dirty[s, r, i, d] = float(value)
        bad[s, r, i] = int(start[s]) + r < lens[s]
    o, lse = kv._attention(c, dirty, start, D ** -0.5)
    _check(o, lse, ref, D, bad)
    # the weights of such a row are NaN where it looks; other heads and positions have theirs
    width = c.width * 16
    scale = D ** -0.5
    score = ops.KvScore(dirty.to(DEV), c.k.to(DEV), c.ks.to(DEV), c.table.to(DEV), start.to(DEV), c.lens.to(DEV), lse,
                        torch.ones(3, 2, width, device=DEV), scale, fmt=fmt).cpu()
    clean = torch.from_numpy(ref["lse"]).float()
    want, added = O.kv_score(q, c.k, c.ks, c.table, start, c.lens, clean, torch.ones(3, 2, width), scale, fmt=fmt)
    nan = np.zeros(want.shape, dtype=bool)
    for s, r, i in np.argwhere(bad):
        nan[s, i // G, :int(start[s]) + r + 1] = True
    assert np.array_equal(np.isnan(score.numpy()), nan)
    dl = (2 * D + 16) * kv.U * ref["ql"].max() + 4 * kv.U * 30 + 2.0 ** -18
    assert (np.abs(score.double().numpy() - want)[~nan] <= (2 * dl * added + 2 * kv.U * np.abs(want))[~nan]).all()
    assert ops.device_status() == 0


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("R,G", [(4, 2), (8, 2), (20, 3)])
def test_a_page_whose_k_scale_is_nan(R, G, D, fmt):
    # rows that see one of its positions are NaN, those before it are not touched
    n = 288 + R // 2  # the last page begins inside the call's rows
    c = kv.Cache([n], 2, D, 16, fmt, seed=203)
    q = kv._rows(1, R, 2 * G, D, seed=204)
    start = c.lens - R
    ref = O.kv_attention(q, *c.host(), c.table, start, c.lens, 0.1, fmt=fmt)
    c.ks[c.table[0, 18].long(), 1] = float("nan")
    bad = np.zeros(q.shape[:3], dtype=bool)
    bad[0, R // 2:, G:] = True
    o, lse = kv._attention(c, q, start, 0.1)
    _check(o, lse, ref, D, bad)
    assert ops.device_status() == 0


@pytest.mark.parametrize("value", ["nan", "inf"])
@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("R,G", [(4, 2), (8, 2), (20, 3)])
def test_a_page_whose_v_scale_is_not_finite(R, G, fmt, value):
    n = 288 + R // 2
    c = kv.Cache([n], 2, 128, 16, fmt, seed=205)
    q = kv._rows(1, R, 2 * G, 128, seed=206)
    start = c.lens - R
    ref = O.kv_attention(q, *c.host(), c.table, start, c.lens, 0.1, fmt=fmt)
    c.vs[c.table[0, 18].long(), 1] = float(value)
    bad = np.zeros(q.shape[:3], dtype=bool)
    bad[0, R // 2:, G:] = True
    o, lse = kv._attention(c, q, start, 0.1)
    _check(o, lse, ref, 128, bad)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("R,G,window,at", [(4, 2, 0, 2), (8, 1, 0, 7), (8, 2, 3, 2), (16, 1, 20, 0), (20, 3, 0, 11),
                                           (30, 1, 20, 3), (130, 2, 0, 64), (150, 1, 40, 60), (40, 1, 0, -200)])
def test_a_nan_among_the_v_codes(R, G, window, at, D):
    # the call's row `at` is the first that sees it: a NaN in o for that row and those after it that still do, and
    # nothing of it in the others'
    c = kv.Cache([300 + R, 40 + R], 2, D, 16, 1, seed=207)
    q = kv._rows(2, R, 2 * G, D, seed=208)
    start = c.lens - R
    ref = O.kv_attention(q, *c.host(), c.table, start, c.lens, 0.1, window=window, sinks=2 if window else 0, fmt=1)
    j = 300 + at
    c.v[c.table[0, j // 16].long(), 1, j % 16, 5] = 0x7F
    o, lse = kv._attention(c, q, start, 0.1, window=window, sinks=2 if window else 0)
    bad = np.zeros(q.shape[:3], dtype=bool)
    bad[0, max(at, 0):(at + window if window else R), G:] = True
    assert bool(o[0, :, G:, 5].cpu()[torch.from_numpy(bad[0, :, G:])].isnan().all())
    o[torch.from_numpy(bad).to(DEV)], lse[torch.from_numpy(bad).to(DEV)] = float("nan"), float("nan")
    _check(o, lse, ref, D, bad)
    assert ops.device_status() == 0


# ---------------------------------------------------------------------------------------------
# page tables
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("entry", [-1, -12345, -2 ** 31, -2 ** 31 + 1, 2 ** 31 - 1])
@pytest.mark.parametrize("R,G", [(1, 2), (1, 16), (1, 20)])
def test_page_numbers_that_the_cache_does_not_have(R, G, entry):
    # the page's positions are left out, whatever the entry's low bits name, and the status word says so
    c = kv.Cache([40], 1, 64, 16, 0, seed=211)
    q = kv._rows(1, 1, G, 64, seed=212)
    start = c.lens - 1
    table = c.table.clone()
    table[0, 1] = entry
    dev = c.dev()
    args = table.to(DEV), start.to(DEV), c.lens.to(DEV)
    ops.device_status()
    o, lse = ops.KvAttention(q.to(DEV), *dev, *args, 0.1)
    assert ops.device_status() == 1 << 8
    idx = np.r_[0:16, 32:40]
    k, v = (O.kv_tokens(x, s, c.table, 0, idx, 0)[:, 0] for x, s in ((c.k, c.ks), (c.v, c.vs)))
    x = q[0, 0].double().numpy() @ k.T * 0.1
    z = np.log(np.exp(x).sum(1))
    p = np.exp(x - z[:, None])
    ref = dict(o=(p @ v)[None, None], lse=z[None, None], av=(p @ np.abs(v))[None, None],
               ql=(np.abs(q[0, 0].double().numpy()) @ np.abs(k).T * 0.1).max(1)[None, None])
    kv._check_attention(o, lse, ref, 64)
    score = ops.KvScore(q.to(DEV), dev[0], dev[2], *args, lse, torch.ones(1, 1, 48, device=DEV), 0.1).cpu()
    assert ops.device_status() == 1 << 8
    want = np.ones(48)
    want[idx] += p.sum(0)
    dl = (2 * 64 + 16) * kv.U * ref["ql"].max() + 4 * kv.U * np.abs(z).max() + 2.0 ** -18
    assert (np.abs(score[0, 0].double().numpy() - want) <= 2 * dl * want + 2 * kv.U * want).all()
    # the other ops leave it out too
    rk, _ = ops.KvRead(*dev, args[0], torch.zeros_like(start).to(DEV), args[2], 40)
    assert ops.device_status() == 1 << 8
    assert not rk[0, 16:32].any() and bool(rk[0, :16].any())


@pytest.mark.parametrize("R,G", [(1, 4), (2, 8), (9, 4)])
def test_tables_of_no_pages(R, G):
    # sequences that hold nothing and a table without columns: nothing to see, nothing to keep
    c = kv.Cache([16, 16], 2, 64, 16, 0, seed=213)
    dev = c.dev()
    table = torch.zeros(2, 0, dtype=torch.int32, device=DEV)
    zero = torch.zeros(2, dtype=torch.int32, device=DEV)
    q = kv._rows(2, R, 2 * G, 64, seed=214).to(DEV)
    o, lse = ops.KvAttention(q, *dev, table, zero, zero, 0.1)
    assert not o.any() and bool(torch.isneginf(lse).all())
    k, v = ops.KvRead(*dev, table, zero, zero, 3)
    assert k.shape == (2, 3, 2, 64) and not k.any() and not v.any()
    score = torch.zeros(2, 2, 0, device=DEV)
    assert ops.KvScore(q, dev[0], dev[2], table, zero, zero, lse, score, 0.1) is score
    new = torch.tensor([[0], [1]], dtype=torch.int32, device=DEV)
    kept, lens, sums = ops.KvEvict(*dev, table, zero, score, new, 5)
    assert bool((kept == -1).all()) and not lens.any() and not sums.any()
    ops.KvAppend(q[:, :, :2], q[:, :, :2], *dev, table, zero, zero)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, c.host()))
    assert ops.device_status() == 0
    # a length that such a table cannot hold is left out
    o, lse = ops.KvAttention(q, *dev, table, zero, zero + 1, 0.1)
    assert ops.device_status() == 1 << 7
    assert not o.any() and bool(torch.isneginf(lse).all())


# ---------------------------------------------------------------------------------------------
# precision
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("small", [2.0 ** -16, 2.0 ** -20, 2.0 ** -22])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("R,G", [(1, 2), (2, 8), (3, 8)])
def test_query_values_far_below_the_rows_largest(R, G, D, small):
    # the largest meets keys of 0 and the others decide
    c = kv.Cache([200], 2, D, 16, 1, seed=221)
    c.k[..., 7] = 0
    q = kv._rows(1, R, 2 * G, D, seed=222).float() * small
    q[..., 7] = 1.0
    q = q.bfloat16()
    start = c.lens - R
    scale = D ** -0.5 / small
    o, lse = kv._attention(c, q, start, scale)
    kv._check_attention(o, lse, O.kv_attention(q, *c.host(), c.table, start, c.lens, scale, fmt=1), D)


# ---------------------------------------------------------------------------------------------
# sizes that take the branches off the common way
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,keep,sinks,recent,kind", [
    (48 * 1024, 30000, 4, 100, "ties"),       # the most whose weights are held in shared memory
    (48 * 1024 + 1, 30000, 4, 100, "ties"),   # ... and one more
    (100003, 777, 0, 0, "even"),
    (100003, 60001, 16, 30000, "special"),
])
def test_evict_of_sequences_longer_than_shared_memory(n, keep, sinks, recent, kind):
    kv.test_evict_matches_the_definition([n, 300], keep, sinks, recent, 1, 64, 256, kind, 0)


@pytest.mark.parametrize("S,R,Hq,Hkv,D,T,fmt,longest,window,sinks", [
    # more than 32 (sequence, row block) pairs, but at most a quarter as many items as blocks
    (40, 1, 4, 1, 128, 32, 0, 5000, 0, 0),
    (70, 2, 8, 1, 64, 16, 1, 4000, 0, 0),
    (33, 2, 8, 1, 128, 16, 1, 3000, 500, 9),
    (37, 3, 8, 1, 128, 64, 0, 3000, 0, 0),     # 24 rows a head
    (34, 20, 1, 1, 64, 16, 0, 5000, 1000, 4),
    (3, 1500, 1, 1, 64, 16, 0, 6000, 0, 0),    # 12 row blocks a sequence
])
def test_many_sequences_of_one_head(S, R, Hq, Hkv, D, T, fmt, longest, window, sinks):
    kv.test_long_items(S, R, Hq, Hkv, D, T, fmt, longest, window, sinks)
