"""The engine with its streams' keys and values in 4 bits (store_bits=4) against the machine put together from the
engine's own banks and the store's formulas in plain Python, bit for bit; and against itself, where one run of many rows has
to equal the same rows one by one."""
import numpy as np
import pytest

import store_reference as ref

pytestmark = pytest.mark.gpu
V = 50257


def layers(M, n):
    """The first n layers of a converted machine."""
    return {k: v for k, v in M.items() if not any(k.startswith(b) and int(k.split(".")[1]) >= n for b in ("qkv.", "proj.", "fc.", "mproj.", "ln1.", "ln2."))}


@pytest.fixture(scope="module")
def eng(M):
    from streaming_machine_b200 import engine
    e = engine.Engine(layers(M, 2), n_streams=2, max_ctx=64, store_bits=4)
    yield e
    e.close()


@pytest.fixture(scope="module")
def peng(PM):
    from streaming_machine_b200 import engine
    e = engine.Engine(layers(PM, 2), n_streams=2, max_ctx=64, store_bits=4)
    yield e
    e.close()


def shape(e, n, ctx):
    if (e.n_streams, e.max_ctx) != (n, ctx):
        e.alloc_streams(n, ctx)
    return e


def heads(X):
    return X.reshape(len(X), 12, 64)


class Gpt2:
    """base2.py:102-114 over the 4-bit store: rows of several streams at once, each stream's rows in order."""

    def __init__(self, e, M):
        self.e, self.M, self.st = e, M, ref.Store({k: M[k] for k in ("arrival", "log2", "exp2")}, 12)

    def rows(self, toks, pos, cu):
        e, M = self.e, self.M
        at = np.array([p for _, p, _ in ref.Store.places(pos, cu)])
        R = M["wte"][np.asarray(toks)].astype(np.int64) + M["wpe"][at].astype(np.int64)
        for l in range(2):
            qkv = e.bank(f"qkv.{l}", R, 0)
            q, k, v = (heads(qkv[:, i * 768:(i + 1) * 768]) for i in range(3))
            self.st.write(k, v, pos, cu, l)
            R = R + e.bank(f"proj.{l}", self.st.attend(q, pos, cu, layer=l).reshape(len(R), 768), 2)
            R = R + e.bank(f"mproj.{l}", e.bank(f"fc.{l}", R, 1), 2)
        return e.bank("head", R, 0)


class Pythia(Gpt2):
    """pythia_base2.py:161-169 over the 4-bit store: both norms of R, the turn before the store, the branches added."""

    def rows(self, toks, pos, cu):
        e, M = self.e, self.M
        at = np.array([p for _, p, _ in ref.Store.places(pos, cu)])
        w, x = M["embed.w"][np.asarray(toks)].astype(np.int64), M["embed.e"].reshape(-1)[np.asarray(toks)].astype(np.int64)[:, None] + 16
        R = np.where(x >= 0, w << np.maximum(x, 0), (w + (1 << np.maximum(-x - 1, 0))) >> np.maximum(-x, 0))
        c, s = (M[k].astype(np.int64)[at][:, None, :] for k in ("cos", "sin"))
        turn = lambda y: np.concatenate([(y[..., :8] * c - y[..., 8:16] * s + (1 << 29)) >> 30,  # noqa: E731
                                         (y[..., 8:16] * c + y[..., :8] * s + (1 << 29)) >> 30, y[..., 16:]], -1)
        for l in range(2):
            qkv = e.bank(f"qkv.{l}", e.gauge(f"ln1.{l}", R), 2).reshape(len(R), 12, 192)
            q, k, v = turn(qkv[..., :64]), turn(qkv[..., 64:128]), qkv[..., 128:]
            self.st.write(k, v, pos, cu, l)
            a = e.bank(f"proj.{l}", self.st.attend(q, pos, cu, layer=l).reshape(len(R), 768), 2)
            R = R + a + e.bank(f"mproj.{l}", e.bank(f"fc.{l}", e.gauge(f"ln2.{l}", R), 3), 2)
        return e.bank("head", e.gauge("lnf", R), 2)


@pytest.mark.parametrize("kind", ["gpt2", "pythia"])
@pytest.mark.parametrize("lens", [[9], [5, 17], [3, 1, 8]])
def test_prompts_and_steps(kind, lens, eng, peng, M, PM):
    e, model, machine = (eng, M, Gpt2) if kind == "gpt2" else (peng, PM, Pythia)
    e = shape(e, len(lens), 64)
    rng = np.random.default_rng(sum(lens))
    prompts = [rng.integers(0, V, n).tolist() for n in lens]
    want = machine(e, model)
    cu = np.concatenate([[0], np.cumsum(lens)])
    lg = want.rows(np.concatenate(prompts), [0] * len(lens), cu)[cu[1:] - 1]
    words, got = e.prefill(prompts, logits=True)
    assert np.array_equal(got, lg) and np.array_equal(words, lg.argmax(1))
    at = np.array(lens)
    for t in range(3):
        lg = want.rows(words, at, None)
        given = words if t == 1 else None                          # fed back on the device, and given
        words, got = e.step(given, n=len(lens), logits=True)
        assert np.array_equal(got, lg) and np.array_equal(words, lg.argmax(1))
        at = at + 1


@pytest.mark.parametrize("n", [1, 2, 3, 33, 64, 70])
@pytest.mark.parametrize("kind", ["gpt2", "pythia"])
def test_steps_equal_the_prompt_pass(kind, n, eng, peng):
    """Streams brought to a length by the prompt pass, and by a shorter prompt and decode steps of the same words, give the
    same scores: the many-row and the few-row arrival, every decode path, more rows than a chunk of the prompt pass."""
    e = shape(eng if kind == "gpt2" else peng, n, 96)
    rng = np.random.default_rng(n)
    ids = rng.integers(0, V, (n, 80))
    lens = rng.integers(60, 81, n)
    _, want = e.prefill([ids[s, :lens[s]] for s in range(n)], logits=True)
    e.prefill([ids[s, :lens[s] - 4] for s in range(n)])
    for t in range(4):
        _, got = e.step([ids[s, lens[s] - 4 + t] for s in range(n)], logits=True)
    assert np.array_equal(got, want)
    # truncated and stepped again: the same, and the generated words are the races' words
    e.rewind(lens - 2, [ids[s, lens[s] - 2] for s in range(n)])
    e.step(logits=True)
    _, again = e.step([ids[s, lens[s] - 1] for s in range(n)], logits=True)
    assert np.array_equal(again, want)
    words = e.generate([ids[s, :lens[s]] for s in range(n)], 3)
    assert np.array_equal(words[:, 0], want.argmax(1))


def test_whole_model(M):
    """All 12 layers: prompts over more than one chunk equal their steps, and a captured step replays."""
    from streaming_machine_b200 import engine
    e = engine.Engine(M, n_streams=5, max_ctx=640, store_bits=4)
    try:
        rng = np.random.default_rng(12)
        ids = rng.integers(0, V, (5, 600))
        lens = [600, 431, 577, 512, 64]
        _, want = e.prefill([ids[s, :lens[s]] for s in range(5)], logits=True)
        e.prefill([ids[s, :lens[s] - 2] for s in range(5)])
        for t in (2, 1):
            _, got = e.step([ids[s, lens[s] - t] for s in range(5)], logits=True)
        assert np.array_equal(got, want)
    finally:
        e.close()


def test_the_16_bit_store_comes_back(eng, M, orc):
    """store_bits is a setting of the next alloc_streams: 4, then 16 again, which is the reference machine bit for bit."""
    from streaming_machine_b200 import engine
    ids = np.random.default_rng(13).integers(0, V, (3, 12))
    e = engine.Engine(M, n_streams=3, max_ctx=32, store_bits=4)
    try:
        four = e.generate(ids, 4)
        e._call("b2_set_scalar", e.h, b"store_bits", 16)
        assert np.array_equal(e.generate(ids, 4), four)            # nothing changes before alloc_streams
        e.alloc_streams(3, 32)
        assert np.array_equal(e.generate(ids, 4), orc.generate(ids, 4))
    finally:
        e.close()


def test_refusals_and_context(eng, M):
    from streaming_machine_b200 import engine
    e = shape(eng, 2, 64)
    for name, v in ((b"store_bits", 8), (b"store_bits", 0), (b"entry_tables", 1)):
        with pytest.raises(engine.B2Error) as ex:
            e._call("b2_set_scalar", e.h, name, v)
        assert ex.value.code == 1
    small = layers(M, 1)
    with pytest.raises(engine.B2Error) as ex:
        engine.Engine(small, max_ctx=32, arrival="float", store_bits=4)
    assert ex.value.code == 1
    with pytest.raises(engine.B2Error) as ex:
        engine.Engine(dict(small, arrival=np.array([1 << 26, 1])), max_ctx=32, store_bits=4)
    assert ex.value.code == 5
    ids = np.random.default_rng(14).integers(0, V, (2, 63))
    e.prefill(ids)
    e.step()                                                       # position 63, the last
    with pytest.raises(engine.B2Error) as ex:
        e.step()
    assert ex.value.code == 4
    assert e.prefill(ids).shape == (2,)                            # and the handle goes on


@pytest.mark.parametrize("switch", [dict(gauge="float"), dict(edge="float")])
def test_beside_float_stages(M, switch):
    """The stage switches that leave the arrival whole: a prompt pass equals its steps (the CUDA-core banks' path)."""
    from streaming_machine_b200 import engine
    e = engine.Engine(layers(M, 1), n_streams=2, max_ctx=48, store_bits=4, **switch)
    try:
        ids = np.random.default_rng(15).integers(0, V, (2, 30))
        _, want = e.prefill(ids, logits=True)
        e.prefill(ids[:, :28])
        for t in (28, 29):
            _, got = e.step(ids[:, t], logits=True)
        assert np.array_equal(got, want)
    finally:
        e.close()


@pytest.mark.parametrize("kind", ["gpt2", "pythia"])
def test_profiled_steps(kind, eng, peng):
    """b2_profile's modes count the store's launches in their classes and change no words."""
    e = shape(eng if kind == "gpt2" else peng, 2, 64)
    ids = np.random.default_rng(16).integers(0, V, (2, 20))
    want = e.generate(ids, 4)
    for mode in (0, 1, 2):
        e._call("b2_profile", e.h, mode)
        assert np.array_equal(e.generate(ids, 4), want)
        _, classes = e.profile_read()
        assert classes["attend"][0] == 4 * 2                       # the prompt pass and three steps of two layers
        assert classes["heads"][0] == 2 * (2 if kind == "pythia" else 1)   # the prompt pass's write (and turn)
        if mode:
            assert classes["attend"][1] > 0
    e._call("b2_profile", e.h, 0)


def test_launch_shapes_of_the_decode_paths(M):
    """The switches of the decode path give the same words over the 4-bit store."""
    import os
    from streaming_machine_b200 import engine
    ids = np.random.default_rng(17).integers(0, V, (3, 20))
    got = []
    for env in ({}, {"B2_WQ": "0"}, {"B2_GRAPH": "0"}, {"B2_PDL": "0"}, {"B2_FUSE_HEADS": "0"}):
        os.environ.update(env)
        try:
            e = engine.Engine(layers(M, 2), n_streams=3, max_ctx=48, store_bits=4)
        finally:
            for k in env:
                del os.environ[k]
        got.append(e.generate(ids, 6))
        e.close()
    assert all(np.array_equal(g, got[0]) for g in got)


@pytest.mark.parametrize("early", ["1", "0"])
@pytest.mark.parametrize("kind,n,ctx", [("gpt2", 1, 1024), ("gpt2", 3, 1024), ("gpt2", 16, 1024), ("gpt2", 64, 1024), ("pythia", 1, 2048),
                                        ("pythia", 16, 2048), ("pythia", 64, 2048)])
def test_long_steps_equal_the_prompt_pass(kind, n, ctx, early, M, PM, monkeypatch):
    """Captured decode steps near a long context's end, with what is held asked for ahead of the dependency wait and without
    (B2_EARLY_KEYS): keys split over clusters of 8, 4 and 2 CTAs, 4 and 8 warps a CTA, registers and ring. The same scores as
    a prompt pass over the same words, over the edges of blocks of 32 positions, and again after a rewind."""
    from streaming_machine_b200 import engine
    monkeypatch.setenv("B2_EARLY_KEYS", early)
    e = engine.Engine(layers(M if kind == "gpt2" else PM, 2), n_streams=n, max_ctx=ctx, store_bits=4)
    try:
        rng = np.random.default_rng(n + ctx)
        ids = rng.integers(0, V, (n, ctx))
        lens = ctx - rng.integers(0, 40, n)
        lens[0] = ctx                                              # the last position
        _, want = e.prefill([ids[s, :lens[s]] for s in range(n)], logits=True)
        e.prefill([ids[s, :lens[s] - 5] for s in range(n)])
        for again in range(2):
            for t in range(5, 0, -1):
                _, got = e.step([ids[s, lens[s] - t] for s in range(n)], logits=True)
            assert np.array_equal(got, want)
            e.rewind(lens - 5, [ids[s, lens[s] - 5] for s in range(n)])
    finally:
        e.close()
