"""The 8-bit key/value cache operators as a decode loop uses them, in plain torch and through the framework.

Five operators work on one paged cache, u8 [pages, Hkv, T, D] for K and for V, with an f32 scale for
each page and head ([pages, Hkv]) and a table of each sequence's pages ([S, width]):

  append     KvAppend: quantise new K/V rows into their pages (the step or prompt before the attention)
  attention  KvAttention: new query rows over the cached tokens, causal, with a sliding window and sinks
  score      KvScore: add each cached token's attention weight to its running sum
  evict      KvEvict: keep the tokens of the largest sums, in pages of their own
  KvRead     the values that the pages hold, bf16 (what append and evict cases return of them)

A code c of a page with scale s stands for s * (c - 128) (fmt int8) or s * e4m3(c) (fmt e4m3).  New
row r of sequence s is position start[s] + r and exists while that is below lens[s]; it sees the
positions j <= start[s] + r with, under a window w, j > start[s] + r - w or j < sinks.

``own`` false computes the plain form: fp32 whatever the inputs' type, rounded once at the end.
"""
import math

import torch

own = False

_QMAX = {"int8": 127.0, "e4m3": 448.0}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _case(name, op, S, Hkv, D, T, len, R=1, Hq=0, fmt="int8", window=0, sinks=0, keep=0, recent=0, ragged=False):
    c = dict(op=op, S=S, R=R, Hq=Hq or Hkv, Hkv=Hkv, D=D, T=T, len=len, fmt=fmt, window=window, sinks=sinks,
             keep=keep, recent=recent, ragged=ragged)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user's next token early in a conversation: the latency of the call
        _case("attention_token_short", "attention", S=1, Hq=32, Hkv=2, D=128, T=16, len=777),
        # one user's next token at the end of a long document: one long axis, few rows
        _case("attention_token_long", "attention", S=1, Hq=32, Hkv=2, D=128, T=64, len=131001),
        # a serving batch of single tokens, each sequence with its own length, one slot idle
        _case("attention_batch", "attention", S=64, Hq=32, Hkv=8, D=128, T=32, len=8192, ragged=True),
        # eight drafted tokens a sequence verified at once
        _case("attention_verify", "attention", S=8, R=8, Hq=32, Hkv=2, D=128, T=64, len=16384, ragged=True),
        # a window layer with sinks: long sequences of which little is read
        _case("attention_window", "attention", S=48, R=3, Hq=16, Hkv=16, D=64, T=16, len=20000, fmt="e4m3",
              window=1024, sinks=4, ragged=True),
        # a chunk of two prompts behind what is cached of them
        _case("attention_prompt", "attention", S=2, R=1500, Hq=16, Hkv=4, D=128, T=32, len=4000),
        # the step's K and V of a serving batch
        _case("append_step", "append", S=64, Hkv=8, D=128, T=32, len=8192, ragged=True),
        # two whole prompts
        _case("append_prompt", "append", S=2, R=6000, Hkv=8, D=128, T=64, len=6000, fmt="e4m3"),
        # the weights of one long sequence
        _case("score_token", "score", S=1, Hq=32, Hkv=2, D=128, T=32, len=65536),
        # the weights of a batch of verified rows
        _case("score_batch", "score", S=32, R=4, Hq=32, Hkv=8, D=64, T=16, len=8192, fmt="e4m3", ragged=True),
        # one long sequence cut to a budget
        _case("evict_long", "evict", S=1, Hkv=2, D=128, T=32, len=20000, keep=8192, sinks=4, recent=512),
        # a batch cut to a small budget, sequences below it among them
        _case("evict_batch", "evict", S=32, Hkv=8, D=128, T=16, len=4096, keep=1000, sinks=4, recent=128, fmt="e4m3",
              ragged=True),
    ]


def _between(rng, lo, hi):
    """An integer of [lo, hi], even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    top = max(work(c)["bytes"] for c in listed()), max(work(c)["flops"] for c in listed())
    # what the plain form holds of the cache in fp32 stays below the largest listed case's
    held = max(c["S"] * c["len"] * c["Hkv"] * c["D"] for c in listed())
    while True:
        op = rng.choice(["attention", "attention", "attention", "append", "score", "evict"])
        D, T, fmt = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128]), rng.choice(["int8", "e4m3"])
        Hkv, G = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 4, 5, 8, 16])
        S = _between(rng, 1, 64)
        R = rng.choice([1, 1, 1, 2, 3, 4, 5, 6, 7, 8])
        length = _between(rng, 1, 131072)
        keep = sinks = recent = window = 0
        if op == "attention" and rng.random() < 0.2:
            S, R = rng.choice([1, 2, 3]), _between(rng, 16, 1500)
        if op == "append" and rng.random() < 0.5:
            S, R = rng.choice([1, 2, 3]), _between(rng, 16, 6000)
        if op in ("attention", "score") and rng.random() < 0.3:
            window, sinks = _between(rng, 16, 4096), rng.choice([0, 1, 4, 16])
        if op == "evict":
            length, R, G = max(length, 32), 1, 1
            keep = _between(rng, 16, max(16, length * 3 // 4))
            sinks, recent = rng.choice([0, 1, 4]), rng.randrange(0, keep // 2)
        length = max(length, R)
        c = _case(None, op, S=S, R=R, Hq=G * Hkv if op in ("attention", "score") else Hkv, Hkv=Hkv, D=D, T=T,
                  len=length, fmt=fmt, window=window, sinks=sinks, keep=keep, recent=recent,
                  ragged=S > 1 and rng.random() < 0.7)
        w = work(c)
        rows = S * R * c["Hq"] * length if op in ("attention", "score") else 0  # the plain form's logits
        if w["bytes"] <= top[0] and w["flops"] <= top[1] and S * length * Hkv * D <= held and rows <= 2 ** 28:
            return c


def _lens(c):
    """(start, lens) of each sequence; a ragged batch has every length up to `len`, and one idle slot."""
    S, R, L = c["S"], c["R"], c["len"]
    lens = [max(R, L * (s * 37 % S + 1) // S) if c["ragged"] else L for s in range(S)]
    if c["ragged"] and S > 2:
        lens[S // 2] = 0
    return [max(0, n - R) for n in lens], lens


def _seen(pos, c):
    """Number of positions that a row at `pos` sees."""
    w = c["window"]
    return pos + 1 if not w or pos + 1 <= w else w + min(c["sinks"], pos + 1 - w)


def work(c):
    S, R, Hq, Hkv, D, T = (c[k] for k in ("S", "R", "Hq", "Hkv", "D", "T"))
    start, lens = _lens(c)
    pages = sum(-(-n // T) for n in lens)
    if c["op"] in ("attention", "score"):
        # a sequence's tokens are read once for all its rows: those its last row sees and, under a
        # window, those that only its earlier rows see
        tokens = sum(min(n, _seen(n - 1, c) + (R - 1 if c["window"] else 0)) for n in lens if n)
        pairs = sum(_seen(a + r, c) for a, n in zip(start, lens) for r in range(n - a)) * Hq
        rows = S * R * Hq
        if c["op"] == "attention":
            return dict(bytes=tokens * Hkv * 2 * D + pages * (8 * Hkv + 4) + rows * (4 * D + 4), flops=pairs * 4 * D)
        return dict(bytes=tokens * Hkv * (D + 8) + pages * (4 * Hkv + 4) + rows * (2 * D + 4), flops=pairs * 2 * D)
    if c["op"] == "append":
        # bf16 in, codes and scales out; then the codes and the bf16 values of the touched pages
        new = sum(n - a for a, n in zip(start, lens))
        held = sum(n - a // T * T for a, n in zip(start, lens) if n > a)
        return dict(bytes=new * Hkv * D * 2 * 3 + held * Hkv * D * 2 * 3 + pages * 4, flops=new * Hkv * D * 4)
    kept = sum(min(n, c["keep"]) for n in lens)
    # the sums, the kept tokens' codes in and out, their indices and sums; then their bf16 values
    return dict(bytes=Hkv * (sum(lens) * 4 + kept * (4 * D + 8) + kept * 2 * D * 3), flops=kept * Hkv * D * 4)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _codes(n, page, fmt, g):
    """Random pages u8 [n, *page]: normal values on a scale that takes about three deviations."""
    out = torch.empty((n, *page), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // math.prod(page))
    for i in range(0, n, step):
        x = torch.randn((min(step, n - i), *page), generator=g, device="cuda") * (_QMAX[fmt] / 3)
        out[i:i + step] = _encode(x, fmt)
    return out


def prepare(case, seed):
    c = case
    S, R, Hq, Hkv, D, T, fmt = (c[k] for k in ("S", "R", "Hq", "Hkv", "D", "T", "fmt"))
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    start, lens = _lens(c)
    width = -(-c["len"] // T)
    total = sum(-(-n // T) for n in lens)
    fresh = -(-c["keep"] // T) if c["op"] == "evict" else 0
    pool = total + S * fresh + 1  # the last page is nobody's: rows of the tables beyond a sequence's end name it
    # the pages lie in the pool in no order
    perm = torch.randperm(pool - 1, generator=g, device="cuda").int()
    need = torch.tensor([-(-n // T) for n in lens], device="cuda")
    first = need.cumsum(0) - need
    at = torch.arange(width, device="cuda")
    table = torch.where(at < need[:, None], perm[(first[:, None] + at).clamp(max=pool - 2)], pool - 1).int().contiguous()
    st = dict(case=c, table=table, start=torch.tensor(start, dtype=torch.int32, device="cuda"),
              lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    st["k_cache"], st["v_cache"] = (_codes(pool, (Hkv, T, D), fmt, g) for _ in range(2))
    st["k_scale"], st["v_scale"] = ((torch.rand(pool, Hkv, generator=g, device="cuda") + 0.5) * 3 / _QMAX[fmt]
                                    for _ in range(2))
    if c["op"] in ("attention", "score", "append"):
        # q, k and v are parts of the rows of one projection
        x = torch.randn(S, R, (Hq + 2 * Hkv) * D, generator=g, device="cuda").bfloat16()
        st["q"] = x[..., :Hq * D].unflatten(-1, (Hq, D))
        st["k"] = x[..., Hq * D:(Hq + Hkv) * D].unflatten(-1, (Hkv, D))
        st["v"] = x[..., (Hq + Hkv) * D:].unflatten(-1, (Hkv, D))
    if c["op"] == "score":
        st["lse"] = _plain_attention(st, values=False)[1]  # what the attention call before returned
        st["score"] = torch.rand(S, Hkv, width * T, generator=g, device="cuda")
    if c["op"] == "append":
        # the touched pages: from the first row's page on
        st["touched"] = (R + T - 2) // T + 1
        st["floor"] = (st["start"] // T * T).int()
    if c["op"] == "evict":
        # few tokens take most of the weight
        st["score"] = torch.rand(S, Hkv, width * T, generator=g, device="cuda").pow(8)
        st["new_table"] = perm[total:total + S * fresh].view(S, fresh).contiguous()
        st["zero"] = torch.zeros(S, dtype=torch.int32, device="cuda")
    return st


# ---------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------
def _decode(codes, fmt):
    return codes.float() - 128.0 if fmt == "int8" else codes.view(torch.float8_e4m3fn).float()


def _encode(x, fmt):
    """Codes of x (in units of the scale): nearest, ties to even; NaN gives the code of 0."""
    x = torch.where(x.isnan(), 0.0, x).clamp(-_QMAX[fmt], _QMAX[fmt])
    return (x.round() + 128.0).to(torch.uint8) if fmt == "int8" else x.to(torch.float8_e4m3fn).view(torch.uint8)


def _pages(cache, scale, table, fmt):
    """fp32 values [S, Hkv, width * T, D] of the sequences' pages."""
    x = _decode(cache[table.long()], fmt) * scale[table.long()][..., None, None]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_logits(st):
    """(logits [S, Hkv, R, G, L] fp32, mask [S, 1, R, 1, L])"""
    c = st["case"]
    S, R, Hq, Hkv, D = (c[k] for k in ("S", "R", "Hq", "Hkv", "D"))
    k = _pages(st["k_cache"], st["k_scale"], st["table"], c["fmt"])
    q = st["q"].float().view(S, R, Hkv, Hq // Hkv, D).transpose(1, 2).reshape(S, Hkv, -1, D)
    logits = (torch.matmul(q, k.transpose(2, 3)) * D ** -0.5).view(S, Hkv, R, Hq // Hkv, -1)
    j = torch.arange(logits.shape[-1], device=q.device)
    pos = st["start"][:, None] + torch.arange(R, device=q.device)
    n = st["lens"][:, None, None]
    see = (j <= pos[..., None]) & (pos[..., None] < n) & (j < n)
    if c["window"]:
        see &= (j > pos[..., None] - c["window"]) | (j < c["sinks"])
    return logits, see[:, None, :, None]


def _plain_attention(st, values=True):
    c = st["case"]
    S, R, Hq, Hkv, D = (c[k] for k in ("S", "R", "Hq", "Hkv", "D"))
    logits, see = _plain_logits(st)
    logits = logits.masked_fill(~see, float("-inf"))
    m = logits.amax(-1, keepdim=True)
    m = torch.where(m.isinf(), 0.0, m)
    e = torch.exp(logits - m)
    total = e.sum(-1, keepdim=True)
    lse = (m + torch.log(total)).squeeze(-1).transpose(1, 2).reshape(S, R, Hq)
    if not values:
        return None, lse
    v = _pages(st["v_cache"], st["v_scale"], st["table"], c["fmt"])
    o = torch.matmul(e.flatten(2, 3), v).view(S, Hkv, R, Hq // Hkv, D) / torch.where(total > 0, total, 1.0)
    return o.transpose(1, 2).reshape(S, R, Hq, D).bfloat16(), lse


def _plain_score(st):
    c = st["case"]
    S, R, Hq, Hkv = (c[k] for k in ("S", "R", "Hq", "Hkv"))
    logits, see = _plain_logits(st)
    lse = st["lse"].view(S, R, Hkv, Hq // Hkv).transpose(1, 2)[..., None]
    p = torch.where(see, torch.exp(logits - lse), 0.0)
    st["score"] += p.sum((2, 3))
    return st["score"]


def _plain_write(st, cache, scale, x):
    """Quantise the rows x [S, R, Hkv, D] into the pages that they touch."""
    c = st["case"]
    S, R, Hkv, D, T, fmt = (c[k] for k in ("S", "R", "Hkv", "D", "T", "fmt"))
    dev, width, spare = x.device, st["table"].shape[1], cache.shape[0] - 1
    b = st["start"][:, None].long() // T + torch.arange(st["touched"], device=dev)
    used = b * T < st["lens"][:, None]
    used &= (st["start"] < st["lens"])[:, None]
    page = torch.where(used, st["table"].gather(1, b.clamp(max=width - 1)).long(), spare)
    pos = b[..., None] * T + torch.arange(T, device=dev)
    row = pos - st["start"][:, None, None]
    new = (row >= 0) & (pos < st["lens"][:, None, None])
    old = row < 0
    take = row.clamp(0, R - 1).flatten(1)[..., None, None].expand(-1, -1, Hkv, D)
    x = x.gather(1, take).view(S, -1, T, Hkv, D).transpose(2, 3).float()
    new, old = new[:, :, None, :, None], old[:, :, None, :, None]
    amax = torch.where(new & x.isfinite(), x.abs(), 0.0).amax((3, 4))
    before = torch.where(old.any(3).squeeze(-1), scale[page], 0.0)
    after = torch.maximum(before, amax / torch.full_like(amax, _QMAX[fmt]))
    some = (after > 0)[..., None, None]
    unit = torch.where(some, after[..., None, None], 1.0)
    codes = cache[page]
    kept = _encode(_decode(codes, fmt) * torch.where(some, before[..., None, None] / unit, 0.0), fmt)
    codes = torch.where(old, kept, torch.where(new, _encode(torch.where(some, x / unit, 0.0), fmt), codes))
    cache[page] = codes
    scale[page] = after


def _plain_read(cache, scale, table, start, lens, rows, fmt):
    """bf16 values [S, rows, Hkv, D] of the positions from start on, 0 from lens on."""
    T = cache.shape[2]
    pos = start[:, None].long() + torch.arange(rows, device=cache.device)
    page = table.long().gather(1, (pos // T).clamp(max=table.shape[1] - 1))
    x = _decode(cache[page, :, pos % T], fmt) * scale[page][..., None]
    return torch.where((pos < lens[:, None])[..., None, None], x, 0.0).bfloat16()


def _plain_evict(st):
    c = st["case"]
    S, Hkv, D, T, keep, fmt = (c[k] for k in ("S", "Hkv", "D", "T", "keep", "fmt"))
    score, n, spare = st["score"], st["lens"][:, None, None], st["k_cache"].shape[0] - 1
    L, pad = score.shape[-1], -keep % T
    j = torch.arange(max(L, keep), device=score.device)
    rank = torch.nn.functional.pad(score, (0, j.numel() - L))
    rank = torch.where((j < c["sinks"]) | (j >= n - c["recent"]), float("inf"), rank)
    rank = torch.where(j < n, rank, float("-inf"))
    kept = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    some = torch.arange(keep, device=score.device) < n
    kept = torch.where(some, kept, j.numel()).sort(-1).values
    src = torch.where(some, kept, 0)
    sums = torch.where(some, score.gather(-1, src), 0.0)
    page = st["table"].long().gather(1, (src // T).flatten(1)).view(src.shape)
    page = torch.nn.functional.pad(torch.where(some, page, spare), (0, pad), value=spare)
    slot = torch.nn.functional.pad(src % T, (0, pad))
    live = torch.nn.functional.pad(some.expand_as(src), (0, pad))
    head = torch.arange(Hkv, device=score.device)[:, None]
    to = st["new_table"].long()
    empty = ~live.unflatten(-1, (-1, T)).any(-1).any(1)
    to = torch.where(empty, spare, to)
    for cache, scale in ((st["k_cache"], st["k_scale"]), (st["v_cache"], st["v_scale"])):
        before = torch.where(live, scale[page, head], 0.0).unflatten(-1, (-1, T))
        after = before.amax(-1)
        ratio = torch.where(after[..., None] > 0, before / torch.where(after > 0, after, 1.0)[..., None], 0.0)
        codes = _encode(_decode(cache[page, head, slot].unflatten(2, (-1, T)), fmt) * ratio[..., None], fmt)
        cache[to] = codes.transpose(1, 2)
        scale[to] = after.transpose(1, 2)
    return torch.where(some, kept, -1).int(), st["lens"].clamp(max=keep), sums


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_plain(st):
    c = st["case"]
    if c["op"] == "attention":
        o, lse = _plain_attention(st)
        return dict(o=o, lse=lse)
    if c["op"] == "score":
        return dict(score=_plain_score(st))
    table, start, lens, rows = st["table"], st["start"], st["lens"], 0
    if c["op"] == "append":
        _plain_write(st, st["k_cache"], st["k_scale"], st["k"])
        _plain_write(st, st["v_cache"], st["v_scale"], st["v"])
        out, start, rows = {}, st["floor"], st["touched"] * c["T"]
    else:
        kept, lens, sums = _plain_evict(st)
        out, start, table, rows = dict(kept=kept, lens=lens, score=sums), st["zero"], st["new_table"], c["keep"]
    return dict(out, k=_plain_read(st["k_cache"], st["k_scale"], table, start, lens, rows, c["fmt"]),
                v=_plain_read(st["v_cache"], st["v_scale"], table, start, lens, rows, c["fmt"]))


def _run_own(st):
    from nemotron_ops_b200 import ops

    c = st["case"]
    fmt = ops.KV_INT8 if c["fmt"] == "int8" else ops.KV_E4M3
    cache = st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"]
    mask = dict(window=c["window"], sinks=c["sinks"])
    if c["op"] == "attention":
        o, lse = ops.KvAttention(st["q"], *cache, st["table"], st["start"], st["lens"], c["D"] ** -0.5, fmt=fmt,
                                 **mask)
        return dict(o=o, lse=lse)
    if c["op"] == "score":
        return dict(score=ops.KvScore(st["q"], st["k_cache"], st["k_scale"], st["table"], st["start"], st["lens"],
                                      st["lse"], st["score"], c["D"] ** -0.5, fmt=fmt, **mask))
    if c["op"] == "append":
        ops.KvAppend(st["k"], st["v"], *cache, st["table"], st["start"], st["lens"], fmt=fmt)
        k, v = ops.KvRead(*cache, st["table"], st["floor"], st["lens"], st["touched"] * c["T"], fmt=fmt)
        return dict(k=k, v=v)
    kept, lens, sums = ops.KvEvict(*cache, st["table"], st["lens"], st["score"], st["new_table"], c["keep"],
                                   sinks=c["sinks"], recent=c["recent"], fmt=fmt)
    k, v = ops.KvRead(*cache, st["new_table"], st["zero"], lens, c["keep"], fmt=fmt)
    return dict(kept=kept, lens=lens, score=sums, k=k, v=v)


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------------------------
def _value(codes, fmt):
    if fmt == "int8":
        return codes.double() - 128
    x = codes.long()
    e, m = (x >> 3) & 15, (x & 7).double()
    mag = torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * torch.exp2((e - 7).double()))
    return torch.where(x > 127, -mag, mag)


def _nearest(x, fmt):
    """x on the grid of the codes, fp64."""
    if fmt == "int8":
        return x.round().clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return ((x / step).round() * step).clamp(-448, 448)


def _tokens(st, cache, scale, s, idx):
    """fp64 values [n, Hkv, D] and scales [n, Hkv] of sequence s's positions idx."""
    T = cache.shape[2]
    page = st["table"][s].long()[idx // T]
    unit = scale[page].double()
    return _value(cache[page, :, idx % T], st["case"]["fmt"]) * unit[..., None], unit


def exact(case, seed):
    st = prepare(case, seed)
    return {"attention": _exact_attention, "score": _exact_score, "append": _exact_append, "evict": _exact_evict}[
        case["op"]](st, *_lens(case))


def _exact_weights(st, s, h, start, n):
    """fp64 logits [rows, G, n] of kv head h's rows, -inf where a row does not see."""
    c = st["case"]
    G = c["Hq"] // c["Hkv"]
    idx = torch.arange(n, device="cuda")
    k = _tokens(st, st["k_cache"], st["k_scale"], s, idx)[0][:, h]
    q = st["q"][s, :n - start, h * G:(h + 1) * G].double()
    x = torch.einsum("rgd,jd->rgj", q, k) / math.sqrt(c["D"])
    pos = torch.arange(start, n, device="cuda")[:, None]
    hidden = idx > pos
    if c["window"]:
        hidden |= (idx <= pos - c["window"]) & (idx >= c["sinks"])
    return x.masked_fill(hidden[:, None], -math.inf)


def _exact_attention(st, start, lens):
    c = st["case"]
    S, R, Hq, Hkv, D = (c[k] for k in ("S", "R", "Hq", "Hkv", "D"))
    if S * R * Hq * c["len"] * D > 1 << 37:
        return None
    G = Hq // Hkv
    o = torch.zeros(S, R, Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((S, R, Hq), -math.inf, dtype=torch.float64, device="cuda")
    for s in range(S):
        n, rows = lens[s], lens[s] - start[s]
        if not n:
            continue
        v = _tokens(st, st["v_cache"], st["v_scale"], s, torch.arange(n, device="cuda"))[0]
        for h in range(Hkv):
            x = _exact_weights(st, s, h, start[s], n)
            z = torch.logsumexp(x, -1)
            lse[s, :rows, h * G:(h + 1) * G] = z
            o[s, :rows, h * G:(h + 1) * G] = torch.exp(x - z[..., None]) @ v[:, h]
    return dict(o=o, lse=lse)


def _exact_score(st, start, lens):
    out = st["score"].double()
    G = st["case"]["Hq"] // st["case"]["Hkv"]
    for s in range(out.shape[0]):
        for h in range(out.shape[1] if lens[s] else 0):
            z = st["lse"][s, :lens[s] - start[s], h * G:(h + 1) * G].double()
            out[s, h, :lens[s]] += torch.exp(_exact_weights(st, s, h, start[s], lens[s]) - z[..., None]).sum((0, 1))
    return dict(score=out)


def _exact_append(st, start, lens):
    c = st["case"]
    S, T, fmt = c["S"], c["T"], c["fmt"]
    rows = st["touched"] * T
    out = {}
    for name in ("k", "v"):
        got = torch.zeros(S, rows, c["Hkv"], c["D"], dtype=torch.float64, device="cuda")
        cache, scale = st[name + "_cache"], st[name + "_scale"]
        for s in range(S):
            first = start[s] // T * T
            for b in range(first, lens[s] if lens[s] > start[s] else first, T):
                end = min(b + T, lens[s])
                x = st[name][s, max(b, start[s]) - start[s]:end - start[s]].double()
                unit = x.abs().amax((0, 2)) / _QMAX[fmt]
                if b < start[s]:
                    held, was = _tokens(st, cache, scale, s, torch.arange(b, start[s], device="cuda"))
                    unit = torch.maximum(unit, was[0])
                    x = torch.cat([held, x])
                unit = unit[:, None]
                got[s, b - first:end - first] = _nearest(x / unit, fmt) * unit
        out[name] = got
    return out


def _exact_evict(st, start, lens):
    c = st["case"]
    S, Hkv, D, T, keep, fmt = (c[k] for k in ("S", "Hkv", "D", "T", "keep", "fmt"))
    sums = torch.zeros(S, Hkv, keep, dtype=torch.float64, device="cuda")
    out = {x: torch.zeros(S, keep, Hkv, D, dtype=torch.float64, device="cuda") for x in ("k", "v")}
    pad = -keep % T
    for s in range(S):
        n, m = lens[s], min(lens[s], keep)
        if not n:
            continue
        every = torch.arange(n, device="cuda")
        parts = {x: _tokens(st, st[x + "_cache"], st[x + "_scale"], s, every) for x in ("k", "v")}
        for h in range(Hkv):
            idx = every
            if n > keep:
                x = st["score"][s, h, :n].double()
                lo, hi = c["sinks"], n - c["recent"]
                best = lo + x[lo:hi].sort(descending=True, stable=True).indices[:keep - lo - c["recent"]]
                idx = torch.cat([every[:lo], best.sort().values, every[hi:]])
            sums[s, h, :m] = st["score"][s, h, idx].double()
            for x in ("k", "v"):
                val, unit = parts[x][0][idx, h], parts[x][1][idx, h]
                unit = torch.nn.functional.pad(unit, (0, keep + pad - m)).view(-1, T).amax(-1).repeat_interleave(T)[:m]
                out[x][s, :m, h] = _nearest(val / unit[:, None], fmt) * unit[:, None]
    return dict(kept=None, lens=None, score=sums, k=out["k"], v=out["v"])
