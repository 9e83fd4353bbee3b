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


def test_refused_tables_stay_refused(small):
    """A table that 4-bit streams cannot take, given when they exist already: every call that would run over them is refused
    (the banks by themselves are not), until the table is a good one or the streams are allocated with 16 bits."""
    from streaming_machine_b200 import engine
    ids = np.random.default_rng(32).integers(0, V, (2, 20))
    big = np.minimum(small["arrival"] * 4, 1 << 25)
    e, fresh = (engine.Engine(m, n_streams=2, max_ctx=32, store_bits=b) for m, b in ((small, 4), (dict(small, arrival=big), 16)))
    try:
        want = scores(e, ids)
        row = np.arange(768)[None] * 100
        bank = e.bank("proj.0", row, 2)
        for name, bad in (("arrival", big), ("arrival", np.r_[0, small["arrival"]]), ("arrival", np.ones(32769)), ("log2", small["log2"] - 1),
                          ("exp2", small["exp2"] - 1)):
            set_array(e, name, bad)
            e._call("b2_finalize", e.h)
            for call in (lambda: e.prefill(ids), lambda: e.step(n=2), lambda: e.generate_device(2, 2), lambda: e.step_host(ids[:, 0])):
                with pytest.raises(engine.B2Error) as ex:
                    call()
                assert ex.value.code == 5
            assert e.bank("proj.0", row, 2).shape == bank.shape    # (by the table given, where the bank reads it)
            set_array(e, name, small[name])
            e._call("b2_finalize", e.h)
            assert np.array_equal(scores(e, ids), want)
        set_array(e, "arrival", big)
        e._call("b2_set_scalar", e.h, b"store_bits", 16)
        e._call("b2_finalize", e.h)
        with pytest.raises(engine.B2Error) as ex:
            e.prefill(ids)                                         # the streams are those in 4 bits still
        assert ex.value.code == 5
        e.alloc_streams(2, 32)
        assert np.array_equal(scores(e, ids), scores(fresh, ids))
    finally:
        e.close()
        fresh.close()


@pytest.mark.parametrize("n", [100, 32768])
def test_a_table_of_another_length(small, n):
    """4-bit streams that exist already take a shorter or longer arrival table: the launches are sized by the new one."""
    from streaming_machine_b200 import engine
    ids = np.random.default_rng(33).integers(0, V, (2, 500))
    table = np.r_[small["arrival"], np.ones(n, np.int64)][:n]
    e, fresh = (engine.Engine(m, n_streams=2, max_ctx=600, store_bits=4) for m in (small, dict(small, arrival=table)))
    try:
        e.prefill(ids)
        set_array(e, "arrival", table)
        e._call("b2_finalize", e.h)
        assert np.array_equal(scores(e, ids), scores(fresh, ids))
    finally:
        e.close()
        fresh.close()


def test_a_refused_array_leaves_the_verdict(small):
    """What b2_set_array refuses does not replace the table, and does not decide whether the table in place suits 4 bits."""
    from streaming_machine_b200 import engine
    e = engine.Engine(small, n_streams=1, max_ctx=32, store_bits=4)
    try:
        for name, bad in (("log2", np.full(10, -1)), ("exp2", np.zeros(65537)), ("log2", np.full(65536, 2 ** 40))):
            with pytest.raises(engine.B2Error):
                set_array(e, name, bad)
            e.alloc_streams(1, 32)                                 # the good table is there still
        set_array(e, "log2", small["log2"] + 65536)
        with pytest.raises(engine.B2Error):
            set_array(e, "log2", np.ones(10))
        e._call("b2_finalize", e.h)
        with pytest.raises(engine.B2Error) as ex:
            e.alloc_streams(1, 32)                                 # and the bad one
        assert ex.value.code == 5
    finally:
        e.close()


@pytest.mark.parametrize("bits", [16, 4])
def test_streams_are_ready_when_alloc_returns(small, bits):
    """b2_alloc_streams clears what it allocates on the legacy stream, which a caller's stream need not wait for: that is done
    when it returns, however long the legacy stream was busy before."""
    import torch
    from streaming_machine_b200 import engine

    class Busy(engine.Engine):
        def alloc_streams(self, n_streams, max_ctx):
            torch.cuda._sleep(400_000_000)                         # a fifth of a second
            super().alloc_streams(n_streams, max_ctx)
            self.done = torch.cuda.default_stream().query()

    e = Busy(small, n_streams=64, max_ctx=1024, store_bits=bits)
    try:
        assert e.done
    finally:
        e.close()


def test_entry_rows_end_with_their_weights(small):
    """Stored layer-0 rows belong to the weights they were built from: after b2_finalize a captured step does without them until
    b2_alloc_streams builds them anew."""
    from streaming_machine_b200 import engine
    ids = np.random.default_rng(36).integers(0, V, (2, 20))
    e = engine.Engine(small, n_streams=2, max_ctx=32)
    try:
        want = scores(e, ids)
        e.set_entry_tables(True)
        e.alloc_streams(2, 32)
        assert np.array_equal(scores(e, ids), want)
        set_array(e, "phi", small["phi"])
        e._call("b2_finalize", e.h)
        assert np.array_equal(scores(e, ids), want)
        e.alloc_streams(2, 32)
        assert np.array_equal(scores(e, ids), want)
    finally:
        e.close()
