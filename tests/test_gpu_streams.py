"""The context's two streams and what is recorded on them.  Needs a real MI355X (-m gpu)."""
import pytest

from gpu_helpers import *  # noqa: F401,F403

pytestmark = pytest.mark.gpu


def test_both_streams_have_the_default_priority():
    assert pa.context().stream_priorities() == {"compute": 0, "comm": 0, "least": 0, "greatest": 0}


@pytest.mark.parametrize("n_dst,n_src", [(1, 1), (1, 300), (257, 64), (70_000, 200_001)])
def test_a_recorded_scatter_add_starts_from_zero_on_every_replay(n_dst, n_src):
    """pa_scatter_add(zero_first) inside a graph, replayed with other eager work, other sources and a spoiled destination between the
    replays: every replay gives the ordered sums (bit for bit: the sums are in the map's order), destinations without a source 0."""
    import pa_amd._lib as L
    rng = np.random.default_rng(n_dst + n_src)
    dest = rng.integers(0, n_dst + 1, n_src).astype(np.int32)           # 1-based; 0 = skipped
    sc = C.c_void_p()
    L.call("pa_scatter_create", pa.context().h, n_dst, n_src, L.ptr(dest), 1, C.byref(sc))
    w, src, other = pa.DeviceVector(n_dst, 0), pa.DeviceVector(n_src, 0), pa.DeviceVector(n_dst, 0)
    with pa.Graph() as g:
        L.call("pa_scatter_add", sc, w.h, src.h, 1)
    for rep in range(5):
        v = rng.standard_normal(n_src)
        want = np.zeros(n_dst)
        np.add.at(want, dest[dest > 0] - 1, v[dest > 0])                # (unbuffered, in the sources' order)
        src.upload(v)
        w.upload(np.full(n_dst, 1e300 if rep % 2 else np.nan))
        L.call("pa_scatter_add", sc, other.h, src.h, 1)                 # the same, eagerly
        pa.context().sync()
        g.launch()
        pa.context().sync()
        assert np.array_equal(w.download(), want), rep
        assert np.array_equal(other.download(), want), rep
    L.call("pa_scatter_destroy", sc)
