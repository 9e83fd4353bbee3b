"""The key/value store held in 4 bits, measured: writing rows into it (and reading them back), reading a stream's
history, and the arrival (attention) over it.

All numbers are whole, at the stream's scale 2^-16. With rnd(x, s) = x 2^-s rounded to nearest (halves up):

  write   a head's 64 key values are held as 4-bit codes c with one shift for each half of 32: t = the bit length of the
          half's largest magnitude, s = max(t - 3, 0) (at most 44), and at least the larger of the two less 3;
          c = rnd(x, s) kept in [-8, 7]. A head's 64 values: the same with one shift. Magnitudes are kept below 2^47.
  read    c 2^s.
  attend  q15 = rnd(q, u), u = max(bit length - 14, 0); a key's score is q15 . k 2^u at 2^-10, over 8 (the root of the
          head's size), rounded; start = the largest; a = ARR[start - score] (0 past the table), Z = sum a;
          w = rnd(a, 1 + M - s), M = the largest value shift among the visible keys, s the key's; out = power(sum w c,
          65536 (M + 1) - log2fix(Z)). A row with no visible key gives zeros.

Streams lie one behind the other: stream i's rows are cu[i] .. cu[i + 1] - 1, the first of them at position pos[i].
A row sees the positions from max(first[i], its own - window + 1) up to its own (no window: 0)."""
import math

import numpy as np
import torch

own = False

HD = 64
LIM = (1 << 30) - 1        # scores are held between -LIM and LIM
TOP = 1 << 47              # magnitudes are held below this


# ---- the cases ------------------------------------------------------------------------------------------------------
def _case(kind, streams, heads, rows, ctx, window=0, drop=0):
    """rows, ctx: (least, most) of the rows a stream gives to the call, and of the positions it already holds."""
    return {"kind": kind, "streams": streams, "heads": heads, "rows_lo": rows[0], "rows_hi": rows[1], "ctx_lo": ctx[0],
            "ctx_hi": ctx[1], "window": window, "drop": drop}


def listed():
    named = {
        # one decode step's keys and values of 64 streams, one layer: latency counts
        "write step 64": _case("write", 64, 12, (1, 1), (32, 159)),
        # a prompt pass writes whole prompts of mixed length
        "write prompts 32x512": _case("write", 32, 12, (129, 512), (0, 0)),
        # a short conversation taken out of the store (to move it, or to continue it at full width)
        "read tail 37": _case("read", 1, 12, (37, 37), (5, 5)),
        # the histories of 16 long streams taken out at once
        "read 16x1000": _case("read", 16, 12, (700, 1000), (0, 24)),
        # the smallest decode step: one stream just begun
        "attend 1x17": _case("attend", 1, 12, (1, 1), (16, 16)),
        # 64 streams after 32-id prompts and up to 128 words
        "attend 64x160": _case("attend", 64, 12, (1, 1), (32, 159)),
        # 16 streams near a context of 1,024
        "attend 16x1024": _case("attend", 16, 12, (1, 1), (960, 1023)),
        # many streams at short contexts
        "attend 512x192": _case("attend", 512, 12, (1, 1), (64, 191)),
        # few streams that go on for long
        "attend 4x32768": _case("attend", 4, 12, (1, 1), (30000, 32767)),
        # odd sizes, a sliding window, dropped beginnings (one stream has nothing left)
        "attend 7x4999 window": _case("attend", 7, 5, (1, 3), (1, 4996), 1000, 4500),
        # a prompt pass over mixed prompts
        "prompts 32x512": _case("attend", 32, 12, (300, 512), (0, 0)),
        # a chunk of a long prompt on top of what the store already holds
        "chunk 2x256 on 8000": _case("attend", 2, 12, (200, 256), (7000, 8000)),
    }
    return [dict(c, name=n) for n, c in named.items()]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _span(rng, lo, hi):
    """(least, most) with the most spread over [lo, hi]."""
    most = _log(rng, max(lo, 1), hi)
    return (rng.randint(lo, most), most)


def draw(rng):
    kind = rng.choice(["write", "read", "decode", "decode", "prompt", "prompt"])
    heads = rng.choice([1, 3, 4, 5, 8, 12, 12, 16])
    if kind in ("write", "read"):
        streams = _log(rng, 1, 512)
        rows = _span(rng, 1, max(1, min(1024, 125000 // (streams * heads))))
        return _case(kind, streams, heads, rows, _span(rng, 0, 200))
    window = _log(rng, 1, 5000) if rng.random() < 0.25 else 0
    drop = _log(rng, 1, 5000) if rng.random() < 0.25 else 0
    if kind == "decode":
        streams = _log(rng, 1, 512)
        ctx = _span(rng, 0, max(1, min(32768, 1500000 // (streams * heads))))
        return _case("attend", streams, heads, (1, 1), ctx, window, drop)
    streams = _log(rng, 1, 32)
    most = _log(rng, 2, max(2, min(1024, math.isqrt(40000000 // (streams * heads)))))
    ctx = _span(rng, 0, max(1, min(8000, 20000000 // (streams * heads * most))))
    return _case("attend", streams, heads, (rng.randint(1, most), most), ctx, window, drop)


def _spread(lo, hi, n, step):
    return [lo + (i * step + hi - lo) % (hi - lo + 1) for i in range(n)]


def _lengths(case):
    """Rows, held positions and first live position of each stream: by the case alone."""
    n = case["streams"]
    rows = _spread(case["rows_lo"], case["rows_hi"], n, 7919)
    ctx = _spread(case["ctx_lo"], case["ctx_hi"], n, 104729)
    first = [case["drop"] if i % 2 else 0 for i in range(n)]
    return rows, ctx, first


def work(case):
    rows, ctx, first = _lengths(case)
    if case["kind"] == "write":      # 64 keys and 64 values in, 67 bytes held, the values that stand for them back
        return {"bytes": sum(rows) * case["heads"] * (1024 + 67 + 67 + 1024), "flops": 4 * 64 * sum(rows) * case["heads"]}
    if case["kind"] == "read":
        return {"bytes": sum(rows) * case["heads"] * (67 + 1024), "flops": 2 * 64 * sum(rows) * case["heads"]}
    keys = pairs = 0
    for n, p, f in zip(rows, ctx, first):
        w = case["window"]
        lows = [max(f, q - w + 1 if w else 0, 0) for q in (p, p + n - 1)]
        keys += max(0, p + n - min(lows))
        q = np.arange(p, p + n)
        pairs += int(np.maximum(q + 1 - np.maximum(f, q - w + 1 if w else 0).clip(0), 0).sum())
    return {"bytes": case["heads"] * (67 * keys + 1024 * sum(rows)), "flops": 4 * 64 * pairs * case["heads"]}


# ---- the inputs -----------------------------------------------------------------------------------------------------
def _tables():
    """The machine's tables: the arrival's e^-x at 2^24, 10 digits after the point; log2 and 2^x with 16 digits."""
    d = torch.arange(17745, dtype=torch.float64)
    m = torch.arange(65536, dtype=torch.float64) / 65536
    return {"arrival": torch.round(torch.exp(-d / 1024) * 2 ** 24).to(torch.int64),
            "log2": torch.round(torch.log2(1 + m) * 65536).to(torch.int64),
            "exp2": torch.round(torch.exp2(m) * 65536).to(torch.int64)}


def _values(gen, rows, heads, size, loud):
    """Whole numbers at 2^-16 of standard deviation `size`, a few of a head's channels `loud` times larger."""
    x = torch.randn(rows, heads, HD, generator=gen, device=gen.device) * (size * 65536)
    c = torch.rand(1, heads, HD, generator=gen, device=gen.device) < 0.06
    return torch.round(torch.where(c, x * loud, x).double()).to(torch.int64)


def _starts(lens, device):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=device)


def _inputs(case, seed):
    """Everything that a call takes, and the history already in the store (stream i's positions 0 .. held[i] - 1)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, ctx, first = _lengths(case)
    i32 = dict(dtype=torch.int32, device="cuda")
    d = {"case": case, "rows": rows, "cu": _starts(rows, "cuda"), "pos": torch.tensor(ctx, **i32),
         "first": torch.tensor(first, **i32) if case["drop"] else None}
    held = [0] * len(rows) if case["kind"] == "write" else [p + n for p, n in zip(ctx, rows)]
    d["held"], d["held_cu"] = held, _starts(held, "cuda")
    d["hk"] = _values(gen, sum(held), case["heads"], 1.0, 6)
    d["hv"] = _values(gen, sum(held), case["heads"], 0.3, 2)
    if sum(held):                    # a stream's first position holds a small value, as models use it
        d["hv"][d["held_cu"][:-1].long()] >>= 5
    if case["kind"] == "write":
        d["k"], d["v"] = _values(gen, sum(rows), case["heads"], 1.0, 6), _values(gen, sum(rows), case["heads"], 0.3, 2)
    if case["kind"] == "attend":
        d["q"] = _values(gen, sum(rows), case["heads"], 1.5, 2)
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    most = case["rows_hi"] + case["ctx_hi"]
    zero = torch.zeros(case["streams"], dtype=torch.int32, device="cuda")
    t = _tables()
    if own:
        from streaming_machine_b200.store import Store
        d["store"] = Store({k: v.numpy() for k, v in t.items()}, n_streams=case["streams"], max_ctx=most, n_head=case["heads"])
        if d["held_cu"][-1]:
            d["store"].write(d["hk"], d["hv"], zero, cu=d["held_cu"], max_rows=max(d["held"]))
    else:
        d["tables"] = {k: v.cuda() for k, v in t.items()}
        shape = (case["streams"], most, case["heads"])
        new = lambda *more: torch.zeros(shape + more, dtype=torch.int8, device="cuda")  # noqa: E731
        d["store"] = {"k": new(HD), "ks": new(2), "v": new(HD), "vs": new(1)}
        if d["held_cu"][-1]:
            _write(d["store"], d["hk"], d["hv"], zero, d["held_cu"])
    del d["hk"], d["hv"]             # a program keeps the store, not what was written into it
    return d


# ---- the plain form -------------------------------------------------------------------------------------------------
def _bits(x):
    """The bit length of whole numbers below 2^53."""
    return torch.frexp(x.double()).exponent.to(torch.int64)


def _rnd(x, s):
    return torch.where(s > 0, ((x >> (s - 1).clamp(min=0)) + 1) >> 1, x)


def _shift(x):
    """The shift that leaves 4 bits of the values along the last axis (kept as an axis of one)."""
    return (_bits(x.abs().amax(-1, keepdim=True)) - 3).clamp(0, 44)


def _codes(x, s):
    return _rnd(x, s).clamp(-8, 7).to(torch.int8)


def _places(pos, cu, rows):
    """The stream and the position of each row."""
    r = torch.arange(rows, device=cu.device)
    s = torch.searchsorted(cu[1:].long(), r, right=True)
    return s, pos.long()[s] + r - cu.long()[s]


def _write(store, k, v, pos, cu):
    s, p = _places(pos, cu, k.shape[0])
    k, v = k.clamp(-TOP, TOP - 1), v.clamp(-TOP, TOP - 1)
    halves = k.unflatten(-1, (2, HD // 2))
    ks = _shift(halves)
    ks = torch.maximum(ks, ks.amax(-2, keepdim=True) - 3)
    vs = _shift(v)
    store["k"][s, p] = _codes(halves, ks).flatten(-2)
    store["ks"][s, p] = ks.squeeze(-1).to(torch.int8)
    store["v"][s, p] = _codes(v, vs)
    store["vs"][s, p] = vs.to(torch.int8)


def _read(store, pos, cu, rows):
    s, p = _places(pos, cu, rows)
    k = store["k"][s, p].long().unflatten(-1, (2, HD // 2)) << store["ks"][s, p].long().unsqueeze(-1)
    return k.flatten(-2), store["v"][s, p].long() << store["vs"][s, p].long()


def _power(x, F, exp2):
    """x 2^(F / 65536) by the table, rounded once."""
    y, s = x * exp2[F & 65535], 16 - (F >> 16)
    return torch.where(s >= 0, _rnd(y, s.clamp(0, 63)), y << (-s).clamp(0, 63))


def _log2fix(z, log2):
    t = _bits(z) - 1
    return t * 65536 + log2[torch.where(t >= 16, z >> (t - 16).clamp(min=0), z << (16 - t).clamp(min=0)) & 65535]


def _attend(store, tables, q, pos, cu, most, window, first):
    rows, ctx = q.shape[0], store["k"].shape[1]
    s, p = _places(pos, cu, rows)
    i = p - pos.long()[s]                                              # the row's place among its stream's
    n = pos.shape[0]
    q = q.clamp(-TOP, TOP - 1)
    u = (_bits(q.abs().amax(-1, keepdim=True)) - 14).clamp(min=0)
    q15 = torch.zeros((n, most) + q.shape[1:], dtype=torch.float64, device=q.device)
    q15[s, i] = _rnd(q, u).double()
    us = torch.zeros((n, most, q.shape[1], 1), dtype=torch.int64, device=q.device)
    us[s, i] = u
    ks = store["ks"].long()
    S = ks.amax(-1, keepdim=True)                                      # [streams, ctx, heads, 1]
    k8 = (store["k"].long().unflatten(-1, (2, HD // 2)) << (ks - S + 3).unsqueeze(-1)).flatten(-2)
    dot = (q15.transpose(1, 2) @ k8.double().permute(0, 2, 3, 1)).long()   # exact: below 2^53
    r = 28 - us.transpose(1, 2) - S.permute(0, 2, 3, 1)                # [streams, heads, rows, ctx]
    up = (-r).clamp(min=0)
    most_up = LIM >> up.clamp(max=62)
    sc = torch.where(r >= 0, _rnd(dot, r.clamp(min=0)), torch.where(dot.abs() <= most_up, dot << up.clamp(max=30), dot.sign() * LIM))
    at = torch.arange(ctx, device=q.device)
    own_pos = pos.long()[:, None] + torch.arange(most, device=q.device)   # [streams, rows]
    lo = torch.zeros_like(own_pos)
    if window:
        lo = (own_pos - window + 1).clamp(min=0)
    if first is not None:
        lo = torch.maximum(lo, first.long()[:, None])
    seen = ((at >= lo[..., None]) & (at <= own_pos[..., None]))[:, None]   # [streams, 1, rows, ctx]
    start = sc.masked_fill(~seen, -LIM - 1).amax(-1, keepdim=True)
    d = start - sc
    arr = tables["arrival"]
    a = torch.where(seen & (d < arr.shape[0]), arr[d.clamp(0, arr.shape[0] - 1)], 0)
    z = a.sum(-1, keepdim=True)
    vs = store["vs"].long().permute(0, 2, 3, 1)                        # [streams, heads, 1, ctx]
    M = torch.where(seen, vs, 0).amax(-1, keepdim=True)
    w = _rnd(a, 1 + M - torch.where(seen, vs, 0))
    num = (w.double() @ store["v"].double().transpose(1, 2)).long()    # exact: below 2^53
    none = z == 0
    out = _power(num, 65536 * (M + 1) - _log2fix(torch.where(none, 1, z), tables["log2"]), tables["exp2"])
    return torch.where(none, 0, out).transpose(1, 2)[s, i]


def run(state):
    case, st = state["case"], state["store"]
    rows, pos, cu, most = sum(state["rows"]), state["pos"], state["cu"], case["rows_hi"]
    if case["kind"] == "write":
        if own:
            st.write(state["k"], state["v"], pos, cu=cu, max_rows=most)
            return st.read(pos, cu=cu, max_rows=most, rows=rows)
        _write(st, state["k"], state["v"], pos, cu)
        return _read(st, pos, cu, rows)
    if case["kind"] == "read":
        if own:
            return st.read(pos, cu=cu, max_rows=most, rows=rows)
        return _read(st, pos, cu, rows)
    if own:
        return st.attend(state["q"], pos, cu=cu, max_rows=most, window=case["window"], first=state["first"])
    return _attend(st, state["tables"], state["q"], pos, cu, most, case["window"], state["first"])


# ---- the definition, number by number in 64 bits ---------------------------------------------------------------------
def _bit_length(x):
    """Bit lengths of non-negative numpy int64."""
    n = np.zeros(x.shape, np.int64)
    for b in (32, 16, 8, 4, 2, 1):
        big = x >= (np.int64(1) << b)
        n[big] += b
        x = np.where(big, x >> b, x)
    return n + (x > 0)


def _near(x, s):
    """floor(x / 2^s + 1/2): the rounding, with nothing that can overflow at these sizes."""
    return np.where(s > 0, (x + (np.int64(1) << np.maximum(s - 1, 0))) >> s, x)


def _held(x, halves):
    """What the store holds of values [rows, heads, 64]: codes and shifts, each [rows, heads, halves, 64 / halves] or [.., 1]."""
    x = np.clip(x, -TOP, TOP - 1).reshape(x.shape[0], x.shape[1], halves, HD // halves)
    s = np.clip(_bit_length(np.abs(x).max(axis=3, keepdims=True)) - 3, 0, 44)
    s = np.maximum(s, s.max(axis=2, keepdims=True) - 3)
    return np.clip(_near(x, s), -8, 7), s


def exact(case, seed):
    d = _inputs(case, seed)
    host = lambda t: t.cpu().numpy()  # noqa: E731
    if case["kind"] == "write":
        return tuple((c << s).reshape(x.shape) for x, (c, s) in ((x, _held(x, h)) for x, h in ((host(d["k"]), 2), (host(d["v"]), 1))))
    rows, ctx, first = _lengths(case)
    hk, hv, hcu = host(d["hk"]), host(d["hv"]), host(d["held_cu"])
    if case["kind"] == "read":
        take = np.concatenate([np.arange(hcu[i] + ctx[i], hcu[i + 1]) for i in range(len(rows))])
        return tuple((c << s).reshape(len(take), -1, HD) for c, s in (_held(hk[take], 2), _held(hv[take], 1)))
    if work(case)["flops"] > 4e10:
        return None
    T = {k: v.numpy() for k, v in _tables().items()}
    q, out, r0 = host(d["q"]), [], 0
    for i, (n, p0, f) in enumerate(zip(rows, ctx, first)):
        here = slice(hcu[i], hcu[i + 1])
        (kc, ks), (vc, vs) = _held(hk[here], 2), _held(hv[here], 1)
        y = np.zeros((n, case["heads"], HD), np.int64)
        for h in range(case["heads"]):
            qi = np.clip(q[r0:r0 + n, h], -TOP, TOP - 1)
            u = np.maximum(_bit_length(np.abs(qi).max(axis=1)) - 14, 0)
            qn = _near(qi, u[:, None]).astype(np.float64)
            # the halves' own products, put on the scale of the key's lower possible shift
            big = ks[:, h, :, 0].max(axis=1)
            dot = sum((qn[:, g * 32:g * 32 + 32] @ kc[:, h, g].T.astype(np.float64)).astype(np.int64) << (ks[:, h, g, 0] - big + 3) for g in (0, 1))
            e = u[:, None] + big[None, :] - 28
            full = dot.astype(object) if e.max() > 30 else dot
            sc = np.where(e > 0, np.clip(full << np.maximum(e, 0), -LIM, LIM), _near(dot, np.maximum(-e, 0))).astype(np.int64)
            at, me = np.arange(p0 + n)[None, :], (p0 + np.arange(n))[:, None]
            low = np.maximum(f, me - case["window"] + 1 if case["window"] else 0)
            live = (at <= me) & (at >= low)
            some = live.any(axis=1)
            gap = np.where(live, sc, -LIM).max(axis=1)[:, None] - sc
            a = np.where(live & (gap < len(T["arrival"])), T["arrival"][np.clip(gap, 0, len(T["arrival"]) - 1)], 0)
            s = vs[:, h, 0, 0][None, :]
            M = np.where(live, s, 0).max(axis=1)
            w = _near(a, np.where(live, 1 + M[:, None] - s, 1))
            num = (w.astype(np.float64) @ vc[:, h, 0].astype(np.float64)).astype(np.int64)
            Z = np.where(some, a.sum(axis=1), 1)
            t = _bit_length(Z) - 1
            F = 65536 * (M + 1) - (t * 65536 + T["log2"][np.where(t >= 16, Z >> np.maximum(t - 16, 0), Z << np.maximum(16 - t, 0)) & 65535])
            x, sh = num * T["exp2"][F & 65535][:, None], (16 - (F >> 16))[:, None]
            y[:, h] = np.where(some[:, None], np.where(sh >= 0, _near(x, np.maximum(sh, 0)), x << np.maximum(-sh, 0)), 0)
        out.append(y)
        r0 += n
    return np.concatenate(out)
