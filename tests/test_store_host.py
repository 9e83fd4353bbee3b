"""The 4-bit store on the CPU: the formulas' own bounds, the layout's permutation, and every refusal that is made before
anything is launched."""
import ctypes

import numpy as np
import pytest
import torch

import store_reference as ref

RNG = np.random.default_rng(41)


@pytest.mark.parametrize("bits", [0, 1, 3, 4, 5, 17, 31, 46, 47, 48, 60, 62])
def test_held_values_are_near(bits):
    """A held value is off by at most half a step 2^s, or by a whole one where the code 8 does not exist (its 4 bits
    reach 7): |x| < 2^t, s = t - 3, so x 2^-s < 8 rounds to at most 8, which is held as 7, a step away at most."""
    for _ in range(20):
        x = np.array([int(RNG.integers(-(1 << 62), 1 << 62)) >> (62 - bits) if bits else 0 for _ in range(64)], dtype=np.int64)
        for held, read, shifts in ((ref.hold_key(x), ref.read_key, 2), (ref.hold_value(x), ref.read_value, 1)):
            c, s = held
            assert all(-8 <= t <= 7 for t in c)
            step = np.repeat([1 << t for t in s], 32) if shifts == 2 else np.full(64, 1 << s)
            off = np.abs(ref.clamp(x) - read(held))
            assert (2 * off <= step * (1 + (np.array(c) == 7))).all()
            if np.abs(x).max() <= 7:          # a bit length of 3: no shift, and every value is its own code
                assert (off == 0).all()


def test_halves_stay_within_three_digits():
    x = np.zeros(64, np.int64)
    x[3], x[40] = 1 << 30, 5
    _, s = ref.hold_key(x)
    assert s == [28, 25]
    x[3] = 9
    assert ref.hold_key(x)[1] == [1, 0]


def _bare(n_head=3):
    """A Store whose checks run without a GPU: the host logic alone (nothing is launched by a call that is refused)."""
    from streaming_machine_b200 import store
    st = object.__new__(store.Store)
    st.h = None
    st._host(torch, "cpu", 0, 4, 64, n_head, 1)
    return st


def test_rows_are_refused():
    st = _bare()
    good = torch.zeros(5, 3, 64, dtype=torch.int64)
    assert st._rows(good, "k")[1] == 192
    qkv = torch.zeros(5, 9 * 64, dtype=torch.int64)
    p, ld = st._rows(qkv[:, 192:384], "k")
    assert ld == 576 and p == qkv.data_ptr() + 192 * 8
    assert st._rows(qkv[:, 192:384].unflatten(1, (3, 64)), "k")[1] == 576
    assert st._rows(torch.from_numpy(np.zeros((0, 3, 64), np.int64)), "k")[1] == 192      # (strides of zero)
    for bad in (good.to(torch.int32), good.float(), good[:, :2], good.transpose(0, 1), good[..., ::2], good[:, :, :32],
                torch.zeros(5, 3, 128, dtype=torch.int64)[..., ::2], good.view(15, 64), torch.zeros(1, 192, dtype=torch.int64).expand(5, 192),
                np.zeros((5, 3, 64), np.int64)):
        with pytest.raises(ValueError):
            st._rows(bad, "k")


def test_numbers_past_32_bits_stay_large():
    """layer, window, max_rows beyond an int32: what reaches the library is as far out, not the number's lower bits."""
    st = _bare()
    st.h, calls = object(), []

    def call(*a):
        calls.append(a)
        return 0
    st._f_write = st._f_read = st._f_attend = st._f_step = call
    x = torch.zeros(4, 3, 64, dtype=torch.int64)
    pos, cu = torch.zeros(4, dtype=torch.int32), torch.arange(5, dtype=torch.int32)
    big = 2 ** 32
    st.write(x, x, pos, cu=cu, max_rows=big + 1, layer=big)
    assert calls[-1][1] == calls[-1][-2] == 2 ** 31 - 1
    st.read(pos, cu=cu, rows=4, max_rows=big + 1, layer=-big)
    assert calls[-1][1] == -2 ** 31 and calls[-1][6] == 2 ** 31 - 1
    st.attend(x, pos, window=big + 5, layer=big)
    assert calls[-1][1] == calls[-1][-3] == 2 ** 31 - 1
    st.step(x, x, x, pos, window=-big + 5, layer=big + 1)
    assert calls[-1][1] == 2 ** 31 - 1 and calls[-1][-3] == -2 ** 31
    st.attend(x, pos, window=5, layer=1)
    assert calls[-1][1] == 1 and calls[-1][-3] == 5
    st.h = None


def test_tables_are_refused():
    st = _bare()
    pos = torch.zeros(4, dtype=torch.int32)
    cu = torch.zeros(5, dtype=torch.int32)
    assert st._table(pos, None, 4, None)[2:] == (4, 4, 1)
    assert st._table(pos, cu, 9, 3)[2:] == (4, 9, 3)
    for args in ((pos, None, 5, None), (pos, None, 4, 2), (pos, cu, 9, None), (pos, cu[:4], 9, 3), (pos.long(), None, 4, None),
                 (pos[::2], None, 2, None), (pos[None], None, 1, None)):
        with pytest.raises(ValueError):
            st._table(*args)
    with pytest.raises(ValueError):
        st._out(torch.zeros(4, 3, 32, dtype=torch.int64), 4, "out")
    with pytest.raises(ValueError):
        st._out(torch.zeros(4, 3, 128, dtype=torch.int64)[..., :64], 4, "out")
    with pytest.raises(ValueError):
        st.read(pos, cu=cu, max_rows=3)                       # rows goes with cu
    x = torch.zeros(4, 3, 64, dtype=torch.int64)
    for call in (lambda: st.attend(x, pos), lambda: st.write(x, x, pos), lambda: st.read(pos), st.sync):
        with pytest.raises(ValueError, match="closed"):
            call()


def test_create_refuses_before_it_touches_a_device():
    from streaming_machine_b200 import engine
    L = engine.lib()
    t = np.ones(65536, np.int64)
    h = ctypes.c_void_p()

    def create(cfg, arr=t, n=100, log2=t, exp2=t, mem=None):
        ptr = [a.ctypes.data if a is not None else None for a in (arr, log2, exp2)]
        return L.b2_store_create(ctypes.byref(engine.StoreConfig(*cfg)), 0, ptr[0], n, ptr[1], ptr[2], mem, ctypes.byref(h))
    for cfg in ((0, 1, 1, 1), (65536, 1, 1, 1), (1, 0, 1, 1), (1, 1025, 1, 1), (1, 1, 0, 1), (1, 1, 1025, 1), (1, 1, 1, 0),
                (1, 1, 1, 65537), (-1, 1, 1, 1)):
        assert create(cfg) == 1 and not h.value
        assert L.b2_store_size(ctypes.byref(engine.StoreConfig(*cfg)), 100) == -1
    assert create((1, 1, 1, 1), mem=4096 + 16) == 1 and not h.value        # memory that is not 32-byte aligned
    # 67 bytes a position and head (positions in 32s), the error words and the tables
    assert L.b2_store_size(ctypes.byref(engine.StoreConfig(3, 2, 5, 33)), 100) == 3 * 2 * 5 * 64 * 67 + 4 * (4 + 131072 + 100)
    for kw in (dict(arr=None), dict(log2=None), dict(exp2=None), dict(n=0), dict(n=-5), dict(n=32769)):
        assert create((1, 1, 1, 1), **kw) == 1 and not h.value
    for f, args in (("b2_store_write", (0, None, 0, None, 0, None, None, 0, 0, 0, None)),
                    ("b2_store_read", (0, None, None, 0, 0, 0, None, None, None)),
                    ("b2_store_attend", (0, None, 0, None, None, None, 0, 0, 0, 0, None, None)), ("b2_store_sync", ())):
        assert getattr(L, f)(None, *args) == 1
    assert L.b2_store_last_error(None) == b"null store"
    L.b2_store_destroy(None)


def test_the_two_references_agree():
    """FastStore (numpy) against Store (Python's whole numbers)."""
    from streaming_machine_b200 import convert
    T = convert.tables()
    rng = np.random.default_rng(42)
    slow, fast = ref.Store(T, 2), ref.FastStore(T, 2, 1)
    k, v, q = (np.round(rng.standard_normal((30, 2, 64)) * s * 65536 * 2.0 ** rng.integers(-5, 2, (30, 2, 1))).astype(np.int64) for s in (1.0, 0.3, 2.0))
    slow.write(k, v, [0], [0, 30])
    fast.write(0, k, v)
    for window, first in ((0, 0), (7, 0), (0, 12), (9, 25)):
        assert np.array_equal(fast.attend(0, q, 0, window, first), slow.attend(q, [0], [0, 30], window, [first]))


@pytest.mark.parametrize("spread", [0, 1, 3, 4, 7, 20])
def test_the_error_in_bits_of_the_largest(spread):
    """What four bits lose, by bit lengths: with t that of the largest magnitude of a value's 64 dims or a key's half, values
    lose at most 2^(t - 4), and less than 2^(t - 3) where the code is 7 (an eighth of 2^t); a key's half next to a larger one, of bit length
    T, at most 2^(T - 7) where that is more (all of it, 7 bits below)."""
    rng = np.random.default_rng(spread)
    for T in (20, 33, 47):
        for _ in range(20):
            x = np.zeros(64, np.int64)
            for half, t in ((slice(0, 32), T), (slice(32, 64), T - spread)):
                x[half] = rng.integers(-(1 << t) + 1, 1 << t, 32)
                x[half][3] = (1 << t) - 1 - rng.integers(0, 2)               # held as 7
            k, v = ref.hold_key(x), ref.hold_value(x)
            for held, got, parts in ((k, ref.read_key(k), (slice(0, 32), slice(32, 64))), (v, ref.read_value(v), (slice(0, 64),))):
                for part in parts:
                    t = int(np.abs(x[part]).max()).bit_length()
                    seven = np.array(held[0])[part] == 7
                    off = np.abs(x[part] - got[part])
                    most = max(t - 4, T - 7)
                    assert (off[~seven] <= 1 << most).all()
                    assert (off[seven] < 2 << most).all()
                    if spread == 0:
                        assert off.max() > (1 << t) // 16                # a sixteenth does not hold
                    if spread >= 7 and part == slice(32, 64):
                        assert (got[part] == 0).all() or spread == 7


def test_ended_stores_are_freed_once(monkeypatch):
    """Two threads that end stores at once free each of them once, and neither fails because the other took the last."""
    import types
    from streaming_machine_b200 import store
    freed = []
    monkeypatch.setattr(store, "lib", lambda: types.SimpleNamespace(b2_store_destroy=freed.append))

    def torch_with(capturing):
        return types.SimpleNamespace(cuda=types.SimpleNamespace(is_current_stream_capturing=capturing))

    def other_thread():                       # between the look at the list and the taking
        if len(store._ended) == 1:
            freed.append(store._ended.pop()[0])
        return False
    for capturing, left in ((lambda: False, []), (other_thread, []), (lambda: True, [1, 2, 3])):
        freed.clear()
        store._ended[:] = [(1, None), (2, None), (3, None)]
        store._free_ended(torch_with(capturing))
        assert sorted(freed + [h for h, _ in store._ended]) == [1, 2, 3] and [h for h, _ in store._ended] == left
    store._ended.clear()
