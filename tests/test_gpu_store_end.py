"""A store that ends while a graph is captured."""
import gc

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", ["close", "last reference", "collected"])
def test_a_store_may_end_during_a_capture(how):
    """Freeing a store waits for the device, which a capture does not allow: it is put off to the next store that is made or
    closed outside of one. The capture goes on, and its replays are right."""
    import torch
    from streaming_machine_b200 import convert, store
    T = convert.tables()
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v, q = (torch.randint(-2 ** 17, 2 ** 17, (2, 3, 64), dtype=torch.int64, device="cuda", generator=g) for _ in range(3))
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    st, old = (store.Store(T, 2, 33, 3) for _ in range(2))
    old.write(k, v, pos)
    out = torch.zeros(2, 3, 64, dtype=torch.int64, device="cuda")
    want = st.step(q, k, v, pos)
    torch.cuda.synchronize()
    box = [old]
    if how == "collected":
        box.append(box)                                            # a cycle: only the collector ends it
    del old
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st.write(k, v, pos)
        if how == "close":
            box[0].close()
        box = None
        gc.collect()
        st.attend(q, pos, out=out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    before = torch.cuda.memory_allocated()
    more = store.Store(T, 2, 33, 3)                                # gives the ended store's memory back first
    assert torch.cuda.memory_allocated() <= before
    more.close()
    st.sync()
    st.close()
    assert np.array_equal(want.shape, (2, 3, 64))
