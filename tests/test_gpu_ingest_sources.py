"""Where ingest takes host bytes from: pinned store blocks, the pinned buffer that stands in for them, ordinary memory."""
import uuid

import numpy as np
import pyarrow as pa
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def store():
    from raydp_amd.runtime.store import SharedObjectStore
    st = SharedObjectStore(f"/dev/shm/raydp_test_sources_{uuid.uuid4().hex[:8]}", "node-test", create=True, capacity=256 << 20)
    yield st
    st.destroy()


def _table(n, seed):
    r = np.random.default_rng(seed)
    return pa.table({c: pa.array(r.standard_normal(n).astype(np.float32)) for c in "ab"})


def _ingest(tables, **kw):
    from raydp_amd.ops import ingest
    ingest.reset_ingest_stats()
    got = ingest.ingest_columns(tables, ["a", "b"], "cuda", False, **kw).cpu().numpy()
    want = np.concatenate([np.stack([t.column(c).to_numpy() for c in "ab"], 1) for t in tables])
    np.testing.assert_array_equal(got, want)
    return ingest.ingest_stats()


def _stored(store, table):
    oid = uuid.uuid4().hex
    store.put(oid, table)
    found, v = store.get(oid)
    assert found
    return v


def test_ordinary_memory_is_pageable_also_after_a_store_was_read(store):
    n = 40_000
    st = _ingest([_stored(store, _table(n, 1))])
    assert st["dma_pageable_bytes"] == 0 and st["dma_pinned_bytes"] >= 8 * n
    assert st["dma_bounced_bytes"] in (0, st["dma_pinned_bytes"])      # all registered, or none
    st = _ingest([_table(n, 2)])
    assert st["dma_pageable_bytes"] >= 8 * n and st["dma_pinned_bytes"] == st["dma_bounced_bytes"] == 0
    inside, outside = _stored(store, _table(n, 3)), _table(3 * n, 4)
    st = _ingest([inside, outside, inside])
    assert st["dma_pinned_bytes"] >= 16 * n and st["dma_pageable_bytes"] >= 24 * n


def test_a_call_that_fails_midway_leaves_the_next_one_right(store, monkeypatch):
    """The second chunk claims more staging memory than there is, which the native code finds after the first is on its way."""
    from raydp_amd.ops import _hip
    n = 60_000
    blocks = [_stored(store, _table(n, s)) for s in (5, 6)]
    lib = _hip.lib()

    class Claims:
        def __getattr__(self, name):
            return getattr(lib, name)

        def rx_ingest_dma(self, chunks, count, *rest):
            real, chunks[1].bytes = chunks[1].bytes, 1 << 40
            try:
                return lib.rx_ingest_dma(chunks, count, *rest)
            finally:
                chunks[1].bytes = real
    with monkeypatch.context() as m:
        m.setattr(_hip, "lib", Claims)
        with pytest.raises(RuntimeError, match="rx_ingest_dma"):
            _ingest(blocks)
    with torch.cuda.stream(torch.cuda.Stream()):
        _ingest(blocks[::-1])
    _ingest([_stored(store, _table(2_000_000, 7))])            # 16 MB: both halves, several times
