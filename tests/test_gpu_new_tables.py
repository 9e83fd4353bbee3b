"""Banks and tables given anew to an engine whose streams and captured step exist already, and allocations that fail:
what runs afterwards is what a fresh engine of the same settings gives."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
V = 50257


def layers(M, n):
    """The first n layers of a converted machine."""
    return {k: v for k, v in M.items() if not any(k.startswith(b) and int(k.split(".")[1]) >= n for b in ("qkv.", "proj.", "fc.", "mproj.", "ln1.", "ln2."))}


@pytest.fixture(scope="module")
def small(M):
    return layers(M, 1)


def set_array(e, name, values):
    a = np.ascontiguousarray(values, dtype=np.int64)
    e._call("b2_set_array", e.h, name.encode(), a.ctypes.data, a.size)


def set_bank(e, M, name):
    w, x, b = (np.ascontiguousarray(M[f"{name}.{k}"], dtype=t) for k, t in (("w", np.int16), ("e", np.int64), ("b", np.int64)))
    e._call("b2_set_bank", e.h, name.encode(), w.ctypes.data, x.ctypes.data, b.ctypes.data, w.shape[0], w.shape[1])


def scores(e, ids):
    """The scores after a prompt, and after each of two steps fed back on the device."""
    out = [e.prefill(ids, logits=True)[1]]
    return np.stack(out + [e.step(n=len(ids), logits=True)[1] for _ in range(2)])


@pytest.mark.parametrize("bits", [16, 4])
def test_a_captured_step_takes_new_tables(small, bits):
    """A decode step is captured once and replayed: after b2_finalize it has to be captured again, or it would read the
    banks and tables that b2_set_bank and b2_set_array have freed."""
    from streaming_machine_b200 import engine
    ids = np.random.default_rng(31).integers(0, V, (2, 20))
    other = dict(small, arrival=np.maximum(small["arrival"] // 2, 1), **{"qkv.0.w": np.flip(small["qkv.0.w"], 1).copy()})
    e, fresh = (engine.Engine(m, n_streams=2, max_ctx=32, store_bits=bits) for m in (small, other))
    try:
        before, want = scores(e, ids), scores(fresh, ids)
        set_array(e, "arrival", other["arrival"])
        set_bank(e, other, "qkv.0")
        e._call("b2_finalize", e.h)
        assert np.array_equal(scores(e, ids), want)
        assert not np.array_equal(before, want)
    finally:
        e.close()
        fresh.close()


@pytest.mark.parametrize("bits", [16, 4])
def test_a_failed_allocation_frees_nothing_twice(M, small, bits):
    """Streams that do not fit, after streams that did: the old buffers are gone with the failed call, and the next one does
    not free their addresses again, which belong to whoever allocated since (torch and another engine here)."""
    import torch
    from streaming_machine_b200 import engine
    ids = np.random.default_rng(34).integers(0, V, (2, 20))
    m = small if bits == 16 else layers(M, 4)
    e = engine.Engine(m, n_streams=2, max_ctx=32, store_bits=bits)
    other = None
    try:
        want = scores(e, ids)
        with pytest.raises(engine.B2Error) as ex:
            e.alloc_streams(65535, 1024)                           # 16 bits: the keys fit, the values do not; 4: 216 GB
        assert ex.value.code == 3
        with pytest.raises(engine.B2Error) as ex:
            e.prefill(ids)
        assert ex.value.code == 6
        torch.cuda.empty_cache()
        sizes = [k for k in range(12, 29) for _ in range(3)]
        held = [torch.full((2 ** k,), k, dtype=torch.uint8, device="cuda") for k in sizes]
        other = engine.Engine(m, n_streams=2, max_ctx=32, store_bits=bits)
        e.alloc_streams(2, 32)
        assert np.array_equal(scores(e, ids), want) and np.array_equal(scores(other, ids), want)
        assert all(bool((t == k).all()) for t, k in zip(held, sizes))
    finally:
        e.close()
        if other:
            other.close()


@pytest.mark.parametrize("bits", [16, 4])
def test_a_failed_allocation_is_told_once(M, small, bits):
    """Streams that do not fit: B2_ERR_NOMEM, and a smaller allocation right after it is not refused for that error."""
    from streaming_machine_b200 import engine
    e = engine.Engine(small if bits == 16 else layers(M, 4), n_streams=1, max_ctx=32, store_bits=bits)
    try:
        want = scores(e, [[1, 2, 3]])
        for _ in range(2):
            with pytest.raises(engine.B2Error) as ex:
                e.alloc_streams(65535, 1024)                       # 319 GB; in 4 bits and 4 layers 216
            assert ex.value.code == 3
            e.alloc_streams(1, 32)
            assert np.array_equal(scores(e, [[1, 2, 3]]), want)
    finally:
        e.close()


@pytest.mark.parametrize("bits", [16, 4])
def test_a_refused_bank_leaves_the_old_one(small, bits):
    """A bank that b2_set_bank refuses for an exponent, in an engine that runs: the old one stays, its captured step too."""
    from streaming_machine_b200 import engine
    ids = np.random.default_rng(35).integers(0, V, (2, 20))
    e = engine.Engine(small, n_streams=2, max_ctx=32, store_bits=bits)
    try:
        want = scores(e, ids)
        with pytest.raises(engine.B2Error) as ex:
            set_bank(e, dict(small, **{"fc.0.e": np.r_[300, small["fc.0.e"][1:]]}), "fc.0")
        assert ex.value.code == 5
        assert np.array_equal(scores(e, ids), want)
    finally:
        e.close()
