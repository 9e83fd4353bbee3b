"""The 4-bit key/value store on the GPU against the formulas in plain Python (store_reference.py), bit for bit: every
result is a whole number, so the tolerance is zero."""
import os

import numpy as np
import pytest

import store_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    from streaming_machine_b200 import convert
    return convert.tables()


def make(T, streams, ctx, heads, layers=1):
    from streaming_machine_b200 import store
    return store.Store(T, n_streams=streams, max_ctx=ctx, n_head=heads, n_layer=layers), ref.Store(T, heads)


def values(rng, rows, heads, size):
    """Normal values of standard deviation 2^16 size; some channels 8 times larger, some rows of one sign or all zero."""
    x = rng.standard_normal((rows, heads, 64)) * 65536 * size
    x[..., rng.random(64) < 0.06] *= 8
    x *= 2.0 ** rng.integers(-6, 3, (rows, heads, 1))
    x[rng.random((rows, heads)) < 0.03] = 0
    return np.round(x).astype(np.int64)


def dev(a, dtype=None):
    import torch
    return torch.as_tensor(np.ascontiguousarray(a, dtype=dtype)).cuda()


def i32(a):
    return dev(a, np.int32)


ROOM = 16384       # a context, and a bound on a stream's rows, that lead to the kernel for many rows however few there are


def run(T, rng, heads, held, rows, window=0, first=None, size=1.5, layers=1, layer=0):
    """Streams that hold held[i] positions take rows[i] more: written, read back and attended, all against the reference, in a
    store and by a bound that just suffice and by ROOM."""
    n = len(held)
    st, pl = make(T, n, max(h + r for h, r in zip(held, rows)), heads, layers)
    room = make(T, n, ROOM, heads, layers)[0]
    try:
        for lens, pos in ((held, [0] * n), (rows, held)):
            if not sum(lens):
                continue
            cu = np.concatenate([[0], np.cumsum(lens)])
            k, v = values(rng, sum(lens), heads, 1.0), values(rng, sum(lens), heads, 0.3)
            st.write(dev(k), dev(v), i32(pos), cu=i32(cu), max_rows=max(lens), layer=layer)
            room.write(dev(k), dev(v), i32(pos), cu=i32(cu), max_rows=ROOM, layer=layer)
            pl.write(k, v, pos, cu, layer)
        q = values(rng, sum(rows), heads, size)
        got = st.attend(dev(q), i32(held), cu=i32(cu), max_rows=max(rows), window=window, layer=layer,
                        first=None if first is None else i32(first)).cpu().numpy()
        many = room.attend(dev(q), i32(held), cu=i32(cu), max_rows=ROOM, window=window, layer=layer,
                           first=None if first is None else i32(first)).cpu().numpy()
        back = [t.cpu().numpy() for t in st.read(i32(held), cu=i32(cu), max_rows=max(rows), rows=sum(rows), layer=layer)]
        st.sync()
        for b, w in zip(back, pl.read(held, cu, layer)):
            assert np.array_equal(b, w)
        want = pl.attend(q, held, cu, window, first, layer)
        assert np.array_equal(got, want) and np.array_equal(many, want)
        room.sync()
    finally:
        st.close()
        room.close()


@pytest.mark.parametrize("held", [0, 1, 2, 7, 15, 16, 31, 32, 33, 63, 64, 127, 300])
def test_one_row(T, held):
    run(T, np.random.default_rng(held), 2, [held, 0, held // 2], [1, 1, 1])


@pytest.mark.parametrize("rows", [[1, 2, 5], [16, 17, 15], [33, 1, 64], [0, 40, 3], [65, 0, 0]])
def test_many_rows(T, rows):
    run(T, np.random.default_rng(sum(rows)), 2, [0, 9, 70], rows)


@pytest.mark.parametrize("heads", [1, 3, 5])
def test_head_counts(T, heads):
    run(T, np.random.default_rng(heads), heads, [20, 3], [1, 4])


@pytest.mark.parametrize("window", [1, 2, 16, 33, 1000])
@pytest.mark.parametrize("rows", [[1, 1, 1], [20, 3, 1], [70, 21, 1]])
def test_windows(T, window, rows):
    run(T, np.random.default_rng(window), 1, [90, 32, 5], rows, window=window)


def test_dropped_beginnings_and_empty_rows(T):
    """first below, inside and past a stream's rows: the second stream's rows see nothing, the third's first two do not,
    and a negative first is none."""
    run(T, np.random.default_rng(3), 2, [50, 50, 10, 5], [3, 3, 4, 1], first=[17, 53, 12, -7])
    run(T, np.random.default_rng(4), 2, [50, 40], [1, 1], first=[51, 40], window=9)
    run(T, np.random.default_rng(4), 1, [50, 50, 10, 5], [70, 30, 25, 1], first=[97, 81, 12, 6])
    run(T, np.random.default_rng(4), 1, [50, 40], [30, 22], first=[70, 20], window=11)


@pytest.mark.parametrize("size", [2.0 ** -16, 0.01, 40.0, 2.0 ** 20, 2.0 ** 40])
def test_query_sizes(T, size):
    """Scores from zeros to ones that are held at their limit (and weights from all alike to a single one)."""
    run(T, np.random.default_rng(5), 1, [40], [2], size=size)
    run(T, np.random.default_rng(5), 1, [40], [33], size=size)


@pytest.mark.parametrize("ctx", [24, ROOM])
def test_extremes(T, ctx):
    """The largest magnitudes, +-2^63 and around 2^47 among them, and rows of zeros: nothing wraps."""
    rng = np.random.default_rng(6)
    big = np.array([-2 ** 63, 2 ** 63 - 1, -2 ** 47, 2 ** 47 - 1, 2 ** 47, -2 ** 47 - 1, 2 ** 46, 7, -8, 0, 1, 2 ** 31], dtype=np.int64)
    st, pl = make(T, 3, ctx, 2)
    n = 24
    pick = lambda rows, p: np.where(rng.random((rows, 2, 64)) < p, rng.choice(big, (rows, 2, 64)), rng.integers(-9, 9, (rows, 2, 64)))  # noqa: E731
    k, v = pick(3 * n, 0.1), pick(3 * n, 0.05)
    k[5], v[9], k[30:34], v[40:44] = 0, 0, 2 ** 47 - 1, -2 ** 63
    cu, pos = [0, n, 2 * n, 3 * n], [0, 0, 0]
    st.write(dev(k), dev(v), i32(pos), cu=i32(cu), max_rows=n)
    pl.write(k, v, pos, cu)
    for b, w in zip(st.read(i32(pos), cu=i32(cu), max_rows=n, rows=3 * n), pl.read(pos, cu)):
        assert np.array_equal(b.cpu().numpy(), w)
    for p in (0.0, 0.02, 0.5, 1.0):
        q = pick(3 * n, p)
        assert np.array_equal(st.attend(dev(q), i32(pos), cu=i32(cu), max_rows=ctx).cpu().numpy(), pl.attend(q, pos, cu))
        # single rows at the last position too
        q1, p1 = q[:3], [n - 1] * 3
        assert np.array_equal(st.attend(dev(q1), i32(p1)).cpu().numpy(), pl.attend(q1, p1))
    st.sync()
    st.close()


def test_other_tables(T):
    """A table whose entries are equal, one that ends at once and one that starts at 1."""
    rng = np.random.default_rng(7)
    for arr in (np.full(3000, 1 << 24), np.array([1]), np.array([1, 0, 1, 5, 7]), np.array([1 << 24, 255, 1, 0, 3])):
        T2 = dict(T, arrival=arr.astype(np.int64))
        run(T2, rng, 1, [30, 2], [1, 1])
        run(T2, rng, 1, [30, 2], [20, 3])
        run(T2, rng, 1, [30, 2], [40, 3])


def test_layers_and_slots_are_apart(T):
    """What one (slot, layer) holds does not show in another; a stream written again from position 0 starts anew."""
    rng = np.random.default_rng(8)
    st, pl = make(T, 3, 40, 2, layers=3)
    for layer in (2, 0, 1, 0):
        lens = [int(t) for t in rng.integers(1, 30, 3)]
        cu = np.concatenate([[0], np.cumsum(lens)])
        k, v = values(rng, cu[-1], 2, 1.0), values(rng, cu[-1], 2, 0.3)
        st.write(dev(k), dev(v), i32([0, 3, 1]), cu=i32(cu), max_rows=30, layer=layer)
        pl.write(k, v, [0, 3, 1], cu, layer)
    for layer in range(3):
        q = values(rng, 3, 2, 1.5)
        assert np.array_equal(st.attend(dev(q), i32([30, 32, 30]), layer=layer).cpu().numpy(), pl.attend(q, [30, 32, 30], layer=layer))
        cu = [0, 40, 80, 120]
        for b, w in zip(st.read(i32([0, 0, 0]), cu=i32(cu), max_rows=40, rows=120, layer=layer), pl.read([0, 0, 0], cu, layer)):
            assert np.array_equal(b.cpu().numpy(), w)
    st.sync()
    st.close()


@pytest.mark.parametrize("ctx,most", [(50, 6), (ROOM, ROOM)])
@pytest.mark.parametrize("off", [0, 1])
def test_strided_rows_and_rows_left_alone(T, off, ctx, most):
    """Keys, values and queries as slices of a qkv row (also at an odd element), outputs with rows that no stream has: those
    stay as they were, in the call's outputs and in the store."""
    import torch
    rng = np.random.default_rng(9)
    H, d = 2, 128
    st, pl = make(T, 3, ctx, H)
    cu, pos, rows = [0, 4, 4, 9], [2, 0, 0], 12
    qkv = torch.zeros(rows, 3 * d + 5 + off, dtype=torch.int64, device="cuda")
    x = values(rng, rows, 3 * H, 1.0).reshape(rows, 3 * d)
    qkv[:, off:off + 3 * d] = dev(x)
    part = [qkv[:, off + i * d:off + (i + 1) * d] for i in range(3)]
    st.write(part[1], part[2], i32(pos), cu=i32(cu), max_rows=most)
    host = [x[:, i * d:(i + 1) * d].reshape(rows, H, 64) for i in range(3)]
    pl.write(host[1], host[2], pos, cu)
    outs = [torch.full((rows, H, 64), -77, dtype=torch.int64, device="cuda") for _ in range(3)]
    got = st.attend(part[0], i32(pos), cu=i32(cu), max_rows=most, out=outs[0])
    assert got is outs[0]
    st.read(i32(pos), cu=i32(cu), max_rows=most, rows=rows, out=outs[1:])
    want = [pl.attend(host[0], pos, cu), *pl.read(pos, cu)]
    for o, w in zip(outs, want):
        o = o.cpu().numpy()
        assert np.array_equal(o[:9], w) and (o[9:] == -77).all()
    every = st.read(i32([0, 0, 0]), cu=i32([0, 50, 100, 150]), max_rows=50, rows=150)
    for b, w in zip(every, pl.read([0, 0, 0], [0, 50, 100, 150])):
        assert np.array_equal(b.cpu().numpy(), w)
    st.sync()
    st.close()


@pytest.mark.parametrize("ctx,most", [(16, 2), (ROOM, ROOM)])
def test_bad_rows_are_flagged_and_skipped(T, ctx, most):
    """Each device check by itself: the stream concerned is left out, the others are done, and sync() reports it once."""
    import torch
    from streaming_machine_b200 import engine
    rng = np.random.default_rng(10)
    st, pl = make(T, 3, ctx, 1)
    k, v, q = (values(rng, 6, 1, 1.0) for _ in range(3))
    good = [0, 2, 4, 6]
    st.write(dev(k), dev(v), i32([0, 0, 0]), cu=i32(good), max_rows=2)
    pl.write(k, v, [0, 0, 0], good)
    want = pl.attend(q, [0, 0, 0], good)
    k2, v2 = values(rng, 6, 1, 1.0), values(rng, 6, 1, 1.0)
    #       cu, pos, the code, the streams left out
    bad = [([0, 2, 1, 6], [0, 0, 0], 1, (1, 2)), ([0, 2, 4, 7], [0, 0, 0], 1, (2,)), ([-1, 2, 4, 6], [0, 0, 0], 1, (0,)),
           ([0, 2, 4, 6], [ctx - 1, 0, 0], 4, (0,)), ([0, 2, 4, 6], [0, -1, 0], 4, (1,)), ([0, 2, 4, 6], [0, 0, 2 ** 31 - 1], 4, (2,)),
           ([0, 2, 4, 2 ** 31 - 1], [0, 0, 0], 1, (2,)), ([-2 ** 31, 2, 4, 6], [0, 0, 0], 1, (0,))]
    for cu, pos, code, left in bad if most == 2 else bad[1:]:      # (the first is told by the bound)
        out = torch.full((6, 1, 64), -5, dtype=torch.int64, device="cuda")
        st.attend(dev(q), i32(pos), cu=i32(cu), max_rows=most, out=out)
        with pytest.raises(engine.B2Error) as ex:
            st.sync()
        assert ex.value.code == code
        st.sync()                                          # reported once
        out = out.cpu().numpy()
        for s in range(3):
            rows = slice(2 * s, 2 * s + 2)
            assert (out[rows] == -5).all() if s in left else np.array_equal(out[rows], want[rows])
        # a write of the same table leaves those streams as they were (the others get what they already hold)
        kk, vv = k.copy(), v.copy()
        for s in left:
            kk[2 * s:2 * s + 2], vv[2 * s:2 * s + 2] = k2[2 * s:2 * s + 2], v2[2 * s:2 * s + 2]
        st.write(dev(kk), dev(vv), i32(pos), cu=i32(cu), max_rows=most)
        with pytest.raises(engine.B2Error):
            st.sync()
        for b, w in zip(st.read(i32([0, 0, 0]), cu=i32(good), max_rows=2, rows=6), pl.read([0, 0, 0], good)):
            assert np.array_equal(b.cpu().numpy(), w)
    st.sync()
    st.close()


def test_refusals(T):
    """What the host refuses: nothing is launched, the store stays usable."""
    import torch
    from streaming_machine_b200 import engine, store
    with pytest.raises(engine.B2Error) as ex:
        store.Store(dict(T, arrival=np.array([1 << 25])), 1, 16, 1)
    assert ex.value.code == 5 and "arrival" in str(ex.value)
    with pytest.raises(engine.B2Error) as ex:
        store.Store(dict(T, arrival=np.array([0, 5])), 1, 16, 1)
    assert ex.value.code == 5
    with pytest.raises(engine.B2Error) as ex:
        store.Store(T, 1, 65537, 1)
    assert ex.value.code == 1
    with pytest.raises(torch.OutOfMemoryError):
        store.Store(T, 1000, 65536, 12, n_layer=12)              # 632 GB
    st, _ = make(T, 2, 16, 1, layers=2)
    x = torch.zeros(2, 1, 64, dtype=torch.int64, device="cuda")
    pos = i32([0, 0])
    for call in (lambda: st.write(x, x, pos, layer=2), lambda: st.write(x, x, pos, layer=-1),
                 lambda: st.attend(x, pos, window=-1), lambda: st.write(x[:1].expand(3, 1, 64).contiguous(), x[:1].expand(3, 1, 64).contiguous(), i32([0, 0, 0])),
                 lambda: st.attend(x, pos, cu=i32([0, 1, 2]), max_rows=-1), lambda: st.attend(x, pos, cu=i32([0, 1, 2]), max_rows=0),
                 lambda: st.attend(x, i32([]), cu=i32([0]), max_rows=1)):
        with pytest.raises(engine.B2Error) as ex:
            call()
        assert ex.value.code == 1
    for call in (lambda: st.write(x.cpu(), x, pos), lambda: st.write(x, x[:1], pos), lambda: st.attend(x.float(), pos),
                 lambda: st.attend(x, pos.long()), lambda: st.attend(x, pos, first=i32([0])), lambda: st.attend(x, pos, out=x[:1])):
        with pytest.raises(ValueError):
            call()
    empty = torch.zeros(0, 1, 64, dtype=torch.int64, device="cuda")   # nothing to do is no error
    st.write(empty, empty, pos, cu=i32([0, 0, 0]), max_rows=0)
    assert st.attend(empty, pos, cu=i32([0, 0, 0]), max_rows=0).shape == (0, 1, 64)
    assert st.attend(empty, i32([])).shape == (0, 1, 64)
    st.sync()
    st.close()
    with pytest.raises(ValueError):
        st.attend(x, pos)


def test_captured_and_on_another_stream(T):
    """write and attend captured into two graphs on one store and replayed with other inputs and positions, then the same
    on a side stream: each the plain calls' results."""
    import torch
    rng = np.random.default_rng(11)
    H = 2
    st, pl = make(T, 4, 64, H)
    pos = i32([0, 5, 0, 9])
    k, v, q = (dev(values(rng, 4, H, 1.0)) for _ in range(3))
    out = torch.zeros(4, H, 64, dtype=torch.int64, device="cuda")
    st.write(k, v, pos)
    st.attend(q, pos, out=out)                               # the first calls load the kernels
    torch.cuda.synchronize()
    graphs = []
    side = torch.cuda.Stream()
    for step in (lambda: st.write(k, v, pos), lambda: st.attend(q, pos, out=out)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append(g)
    pl.write(k.cpu().numpy(), v.cpu().numpy(), [0, 5, 0, 9])
    at = np.array([0, 5, 0, 9])
    for t in range(3):
        at = at + 1
        pos.copy_(i32(at))
        for x in (k, v, q):
            x.copy_(dev(values(rng, 4, H, 1.0)))
        pl.write(k.cpu().numpy(), v.cpu().numpy(), at)
        if t < 2:
            for g in graphs:
                g.replay()
        else:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                st.write(k, v, pos)
                st.attend(q, pos, out=out)
            side.synchronize()
        assert np.array_equal(out.cpu().numpy(), pl.attend(q.cpu().numpy(), at))
    st.sync()
    st.close()


def run_long(T, rng, heads, held, rows, window=0, first=None, max_rows=None):
    """As run(), for many keys: the numpy reference."""
    n = len(held)
    st = make(T, n, max(h + r for h, r in zip(held, rows)), heads)[0]
    pl = ref.FastStore(T, heads, n)
    try:
        total = [h + r for h, r in zip(held, rows)]
        cu = np.concatenate([[0], np.cumsum(total)])
        k, v = values(rng, cu[-1], heads, 1.0), values(rng, cu[-1], heads, 0.3)
        st.write(dev(k), dev(v), i32([0] * n), cu=i32(cu), max_rows=max(total))
        for s in range(n):
            pl.write(s, k[cu[s]:cu[s + 1]], v[cu[s]:cu[s + 1]])
        cu = np.concatenate([[0], np.cumsum(rows)])
        q = values(rng, cu[-1], heads, 1.5)
        got = st.attend(dev(q), i32(held), cu=i32(cu), max_rows=max_rows or max(rows), window=window,
                        first=None if first is None else i32(first)).cpu().numpy()
        st.sync()
        for s in range(n):
            want = pl.attend(s, q[cu[s]:cu[s + 1]], held[s], window, 0 if first is None else first[s])
            assert np.array_equal(got[cu[s]:cu[s + 1]], want), s
    finally:
        st.close()


@pytest.mark.parametrize("heads,held,rows", [
    (1, [2100, 40], [1, 1]), (12, [1030] * 5 + [3] * 11, [1] * 16), (1, [20000], [1]), (12, [60, 99, 7] * 50, [1] * 150),
    (2, [40000, 33000, 5], [1, 2, 1]), (5, [4100], [20]),
    (12, [199, 60] * 75, [1] * 150), (1, [900, 77] * 50, [1] * 100), (2, [1630, 9] * 25, [1] * 50), (6, [13000] * 3 + [40] * 5, [1] * 8),
    (1, [60001], [1]), (2, [700, 3], [40, 64]), (1, [3000], [130]), (3, [6000, 50], [64, 1]), (12, [2000], [130]),
    (2, [9000], [200]), (1, [30000], [64]), (5, [1500, 700], [100, 40]), (12, [4100, 9], [64, 50]),
    (1, [3] * 1100, ([24, 1, 70] + [2] * 8) * 100), (12, [0] * 8, [200, 130, 64, 65, 127, 128, 1, 30])])
def test_long_and_many(T, heads, held, rows):
    """Every shape of launch: a warp, 4, 8 and 16 warps a row and head, keys split over clusters of 2 to 8 CTAs, for few
    rows and for many; streams much shorter than the longest beside it."""
    run_long(T, np.random.default_rng(len(held) + heads), heads, held, rows)


@pytest.mark.parametrize("rows", [[1, 1], [18, 3], [90, 22], [700, 22]])
def test_long_windows(T, rows):
    run_long(T, np.random.default_rng(16), 2, [3000, 1500], rows, window=1111, first=[0, 1490])


def test_max_rows_is_a_bound(T):
    """A bound that no stream reaches, up to the whole context: the same results by whichever kernel it leads to."""
    for bound in (3, 20, 21, 64, 400):
        run_long(T, np.random.default_rng(17), 2, [390, 0, 100], [2, 3, 1], max_rows=bound)


def test_far_into_memory(T):
    """A store whose arrays pass 2^32 bytes: its last stream's last positions."""
    st, pl = make(T, 256, 65536, 12)
    rng = np.random.default_rng(18)
    pos = np.zeros(256, np.int32)
    cu = np.zeros(257, np.int32)
    pos[255], cu[256] = 65536 - 40, 40
    k, v, q = (values(rng, 40, 12, s) for s in (1.0, 0.3, 1.5))
    st.write(dev(k), dev(v), i32(pos), cu=i32(cu), max_rows=40)
    got = st.attend(dev(q), i32(pos), cu=i32(cu), max_rows=40, window=9)
    one = pos.copy()
    one[255] = 65535
    cu1 = np.minimum(cu, 1)
    last = st.attend(dev(q[39:]), i32(one), cu=i32(cu1), max_rows=1, window=9)
    back = st.read(i32(pos), cu=i32(cu), max_rows=40, rows=40)
    st.sync()
    st.close()
    for s in (slice(0, 2),):                                       # two heads of the twelve, by the slow reference
        pl.H = 2
        pl.write(k[:, s], v[:, s], [65536 - 40], [0, 40])
        want = pl.attend(q[:, s], [65536 - 40], [0, 40], window=9)
        assert np.array_equal(got[9:, s].cpu().numpy(), want[9:]) and np.array_equal(last[:, s].cpu().numpy(), want[39:])
        for b, w in zip(back, pl.read([65536 - 40], [0, 40])):
            assert np.array_equal(b[:, s].cpu().numpy(), w)


def test_out_may_be_the_queries(T):
    import torch
    for rows in ([1, 1], [25, 70]):
        rng = np.random.default_rng(19)
        st, _ = make(T, 2, 200, 3)
        cu = np.concatenate([[0], np.cumsum(rows)])
        hist = [dev(values(rng, 400, 3, s)) for s in (1.0, 0.3)]
        st.write(*hist, i32([0, 0]), cu=i32([0, 200, 400]), max_rows=200)
        q = dev(values(rng, cu[-1], 3, 1.5))
        want = st.attend(q, i32([100, 130]), cu=i32(cu), max_rows=max(rows))
        assert st.attend(q, i32([100, 130]), cu=i32(cu), max_rows=max(rows), out=q) is q
        assert torch.equal(q, want)
        st.sync()
        st.close()


def test_calls_at_once(T):
    """Two streams of work on one store (readers of one half of the slots, a writer of the other), many times over."""
    import torch
    rng = np.random.default_rng(20)
    st, _ = make(T, 4, 700, 4)
    hist = [dev(values(rng, 4 * 600, 4, s)) for s in (1.0, 0.3)]
    cu = i32([0, 600, 1200, 1800, 2400])
    st.write(*hist, i32([0] * 4), cu=cu, max_rows=600)
    q1, q2 = dev(values(rng, 2, 4, 1.5)), dev(values(rng, 100, 4, 1.5))
    args1, args2 = (i32([599, 400]),), (i32([550, 550]),)
    cu2 = i32([0, 50, 100])
    want1, want2 = st.attend(q1, *args1), st.attend(q2, *args2, cu=cu2, max_rows=50)
    # the writer rewrites the positions 600 .. 649 of all four: nobody reads those
    more = [dev(values(rng, 200, 4, s)) for s in (1.0, 0.3)]
    cuw, posw = i32([0, 50, 100, 150, 200]), i32([600] * 4)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(30):
        with torch.cuda.stream(streams[0]):
            got.append((want1, st.attend(q1, *args1)))
        with torch.cuda.stream(streams[1]):
            got.append((want2, st.attend(q2, *args2, cu=cu2, max_rows=50)))
        with torch.cuda.stream(streams[2]):
            st.write(*more, posw, cu=cuw, max_rows=50)
    torch.cuda.synchronize()
    assert all(torch.equal(w, g) for w, g in got)
    st.sync()
    st.close()


def test_the_library_allocates(T):
    """The C ABI with memory = NULL: the library's own allocation, and its refusal of one that does not fit."""
    import ctypes
    import torch
    from streaming_machine_b200 import engine, store
    L = engine.lib()
    t = [np.ascontiguousarray(T[k], dtype=np.int64) for k in ("arrival", "log2", "exp2")]

    def create(*cfg):
        h = ctypes.c_void_p()
        rc = L.b2_store_create(ctypes.byref(engine.StoreConfig(*cfg)), 0, t[0].ctypes.data, t[0].size, t[1].ctypes.data,
                               t[2].ctypes.data, None, ctypes.byref(h))
        return rc, h
    rc, h = create(1000, 12, 12, 65536)
    assert rc == 3 and b"cudaMalloc" in L.b2_store_last_error(h)
    assert L.b2_store_sync(h) == 1                             # a store that was not made refuses every call
    L.b2_store_destroy(h)
    rc, h = create(2, 1, 3, 40)
    assert rc == 0
    rng = np.random.default_rng(21)
    k, v, q = (dev(values(rng, 2, 3, s)) for s in (1.0, 0.3, 1.5))
    pos, out = i32([0, 0]), torch.zeros(2, 3, 64, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    assert L.b2_store_write(h, 0, k.data_ptr(), 192, v.data_ptr(), 192, None, pos.data_ptr(), 2, 2, 1, None) == 0
    assert L.b2_store_attend(h, 0, q.data_ptr(), 192, None, pos.data_ptr(), None, 2, 2, 1, 0, out.data_ptr(), None) == 0
    assert L.b2_store_sync(h) == 0
    L.b2_store_destroy(h)
    pl = ref.Store(T, 3)
    pl.write(k.cpu().numpy(), v.cpu().numpy(), [0, 0])
    assert np.array_equal(out.cpu().numpy(), pl.attend(q.cpu().numpy(), [0, 0]))


@pytest.mark.parametrize("n,heads,ctx", [(1, 12, 100), (3, 2, 33), (64, 12, 160), (150, 12, 70), (2, 1, 5000), (16, 12, 1040), (1, 1, 30000),
                                         (150, 12, 190), (100, 1, 930), (50, 2, 1650), (1, 1, 60000)])
def test_step_is_write_and_attend(T, n, heads, ctx):
    """step() on one store, write() and attend() on another, token by token at every place in a block of 32 positions, with
    windows and dropped beginnings (that leave a row nothing): the same outputs and the same store."""
    import torch
    rng = np.random.default_rng(n + ctx)
    a, b = make(T, n, ctx, heads)[0], make(T, n, ctx, heads)[0]
    start = max(ctx - 34, 0)
    hist = [dev(values(rng, n * start, heads, s)) for s in (1.0, 0.3)]
    for st in (a, b):
        st.write(*hist, i32([0] * n), cu=i32(np.arange(n + 1) * start), max_rows=start)
    qkv = torch.zeros(n, 3 * heads * 64 + 1, dtype=torch.int64, device="cuda")
    for t in range(min(34, ctx)):
        pos = i32(start + t - rng.integers(0, t + 1, n))
        window = int(rng.choice([0, 0, 1, 40, ctx]))
        first = i32(rng.integers(0, ctx + 4, n)) if t % 3 == 2 else None
        x = values(rng, n, 3 * heads, 1.0)
        if t % 5 == 4:
            x[:, :, 0] = rng.choice([-2 ** 63, 2 ** 46, 2 ** 31, 0], (n, 3 * heads))
        qkv[:, t % 2:t % 2 + 3 * heads * 64] = dev(x.reshape(n, -1))
        q, k, v = (qkv[:, t % 2 + i * heads * 64:t % 2 + (i + 1) * heads * 64] for i in range(3))
        got = a.step(q, k, v, pos, window=window, first=first)
        b.write(k, v, pos)
        assert torch.equal(got, b.attend(q, pos, window=window, first=first)), t
    rows = i32(np.arange(n + 1) * ctx)
    for u, w in zip(a.read(i32([0] * n), cu=rows, max_rows=ctx, rows=n * ctx), b.read(i32([0] * n), cu=rows, max_rows=ctx, rows=n * ctx)):
        assert torch.equal(u, w)
    a.sync()
    b.sync()
    a.close()
    b.close()


@pytest.mark.parametrize("ctx", [100, 5000])
def test_step_out_may_be_an_input(T, ctx):
    """step() into its own q, k or v, rows that see nothing among them: the outputs and the store of a step into new memory."""
    import torch
    rng = np.random.default_rng(ctx)
    pos, first = i32([ctx - 1, 40, 70]), i32([0, 41, 71])
    hist = [dev(values(rng, 3 * (ctx - 1), 12, s)) for s in (1.0, 0.3)]
    x = [dev(values(rng, 3, 12, s)) for s in (1.5, 1.0, 0.3)]
    want = None
    for into in (None, 0, 1, 2):
        st, _ = make(T, 3, ctx, 12)
        st.write(*hist, i32([0] * 3), cu=i32(np.arange(4) * (ctx - 1)), max_rows=ctx - 1)
        args = [t.clone() for t in x]
        y = st.step(*args, pos, first=first, out=None if into is None else args[into])
        held = st.read(i32([0] * 3), cu=i32(np.arange(4) * ctx), max_rows=ctx, rows=3 * ctx)
        st.sync()
        want = want or (y, *held)
        assert all(torch.equal(a, b) for a, b in zip((y, *held), want)), into
        assert int(y[0].abs().max()) > 0 and int(y[1:].abs().max()) == 0
        st.close()


def test_step_refusals_and_flags(T):
    import torch
    from streaming_machine_b200 import engine
    st, _ = make(T, 2, 16, 1)
    x = torch.zeros(2, 1, 64, dtype=torch.int64, device="cuda")
    pos = i32([0, 0])
    for call in (lambda: st.step(x, x, x, pos, layer=1), lambda: st.step(x, x, x, pos, window=-1),
                 lambda: st.step(*[torch.zeros(3, 1, 64, dtype=torch.int64, device="cuda")] * 3, i32([0, 0, 0]))):
        with pytest.raises(engine.B2Error) as ex:
            call()
        assert ex.value.code == 1
    for call in (lambda: st.step(x, x[:1], x, pos), lambda: st.step(x, x, x[:1], pos), lambda: st.step(x, x, x, i32([0]))):
        with pytest.raises(ValueError):
            call()
    st.step(x, x, x, i32([16, 3]))
    with pytest.raises(engine.B2Error) as ex:
        st.sync()
    assert ex.value.code == 4
    empty = torch.zeros(0, 1, 64, dtype=torch.int64, device="cuda")
    assert st.step(empty, empty, empty, i32([])).shape == (0, 1, 64)
    st.sync()
    st.close()


FIRST_CALLS = """
import sys, numpy as np, torch
from streaming_machine_b200 import convert, store
def i32(x): return torch.tensor(x, dtype=torch.int32, device="cuda")
g = torch.Generator(device="cuda").manual_seed(1)
def x(*s): return torch.randint(-2 ** 17, 2 ** 17, s, dtype=torch.int64, device="cuda", generator=g)
st, other = (store.Store(convert.tables(), 3, 96, 2) for _ in range(2))
cu, zero, pos, end = i32([0, 30, 60, 90]), i32([0, 0, 0]), i32([30, 30, 30]), i32([31, 31, 31])
k, v, q = x(90, 2, 64), x(90, 2, 64), x(90, 2, 64)
src = [x(3, 2, 64) for _ in range(3)]
q1, k1, v1 = (torch.zeros_like(s) for s in src)
out = torch.full((3, 2, 64), -7, dtype=torch.int64, device="cuda")
pinned = torch.zeros(90, 2, 64, dtype=torch.int64).pin_memory()
side = torch.cuda.Stream()
torch.cuda.synchronize()
def work(st, capture):
    for a, b in zip((q1, k1, v1), src):
        a.copy_(b)                                           # a copy on the device before
    st.write(k, v, zero, cu=cu, max_rows=30)
    fork = torch.cuda.Event()
    fork.record()
    with torch.cuda.stream(side):                            # two readers at once
        side.wait_event(fork)
        many = st.attend(q, zero, cu=cu, max_rows=30)
        join = torch.cuda.Event()
        join.record()
    few = st.attend(q1, i32_29)
    torch.cuda.current_stream().wait_event(join)
    step = st.step(q1, k1, v1, pos)                          # behind both
    out.zero_()                                              # a fill between two calls
    st.attend(q1, pos, out=out)
    held = st.read(zero, cu=cu, max_rows=30, rows=90)
    pinned.copy_(held[0], non_blocking=True)                 # a copy to the host behind
    return many, few, step, held
i32_29 = i32([29, 29, 29])
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):                                # the process's first calls
    got = work(st, True)
for _ in range(2):
    graph.replay()
torch.cuda.synchronize()
host, o = pinned.clone(), out.clone()
want = work(other, False)
torch.cuda.synchronize()
flat = lambda r: (r[0], r[1], r[2], *r[3])
assert all(torch.equal(a, b) for a, b in zip(flat(got), flat(want)))
assert torch.equal(host, want[3][0].cpu()) and torch.equal(o, out) and torch.equal(out, want[2])
assert not torch.equal(want[1], want[2]) and int(want[2].abs().max()) > 0
st.sync()
other.sync()
print("same")
"""


def test_first_calls_captured_and_forked():
    """A process's first calls inside a capture, on two streams that part and meet, with copies and fills between them:
    replayed, the plain calls' results."""
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr


def test_a_writer_beside_readers(T):
    """Readers of the positions 0 .. 599 on two streams of work while a third writes the positions from 600 on, other values
    every time: the readers' results do not move, and what was written last is what the store holds and attends over."""
    import torch
    rng = np.random.default_rng(22)
    st, quiet = make(T, 4, 700, 4)[0], make(T, 4, 700, 4)[0]
    hist = [dev(values(rng, 4 * 600, 4, s)) for s in (1.0, 0.3)]
    cu = i32([0, 600, 1200, 1800, 2400])
    for s in (st, quiet):
        s.write(*hist, i32([0] * 4), cu=cu, max_rows=600)
    q1, q2, q3 = dev(values(rng, 4, 4, 1.5)), dev(values(rng, 100, 4, 1.5)), dev(values(rng, 200, 4, 1.5))
    p1, p2, cu2 = i32([599, 400, 599, 31]), i32([550, 550]), i32([0, 50, 100])
    want1, want2 = st.attend(q1, p1), st.attend(q2, p2, cu=cu2, max_rows=50)
    new = [[dev(values(rng, 200, 4, s)) for s in (1.0, 0.3)] for _ in range(31)]
    cuw, posw = i32([0, 50, 100, 150, 200]), i32([600] * 4)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for kv in new:
        with torch.cuda.stream(streams[0]):
            got.append((want1, st.attend(q1, p1)))
        with torch.cuda.stream(streams[1]):
            got.append((want2, st.attend(q2, p2, cu=cu2, max_rows=50)))
        with torch.cuda.stream(streams[2]):
            st.write(*kv, posw, cu=cuw, max_rows=50)
    torch.cuda.synchronize()
    assert all(torch.equal(w, g) for w, g in got)
    quiet.write(*new[-1], posw, cu=cuw, max_rows=50)
    every = dict(cu=i32(np.arange(5) * 650), max_rows=650, rows=2600)
    for a, b in zip(st.read(i32([0] * 4), **every), quiet.read(i32([0] * 4), **every)):
        assert torch.equal(a, b)
    assert torch.equal(st.attend(q3, posw, cu=cuw, max_rows=50), quiet.attend(q3, posw, cu=cuw, max_rows=50))
    for s in (st, quiet):
        s.sync()
        s.close()
