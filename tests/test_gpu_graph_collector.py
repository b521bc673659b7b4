"""Arrays that wait for the garbage collector do not fail a capture."""
import gc

import numpy as np
import pytest

from test_gpu_int8 import T  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


def test_capture_while_the_collector_is_due(T):  # noqa: F811
    rng = np.random.default_rng(0)
    w, x = (T.to_device(rng.standard_normal(s).astype(np.float32)) for s in ((64, 32), (10, 32)))
    want = T.mul_mat(w, x).numpy()
    st, out = T.Stream(), T.empty((10, 64))
    T.mul_mat(w, x, out=out, stream=st)
    st.synchronize()

    def work():
        made = []
        for _ in range(1000):                                  # (many containers: past the threshold)
            made.append([made])
        T.mul_mat(w, x, out=out, stream=st)

    before = gc.get_threshold()
    held = [T.to_device(np.zeros(8, np.float32))]
    held.append(held)
    del held                                                   # a cycle: only the collector frees its array
    gc.set_threshold(50, 1, 1)
    try:
        g = T.Graph(st, work)
    finally:
        gc.set_threshold(*before)
    assert gc.isenabled()
    for _ in range(3):
        g.launch()
        st.synchronize()
        assert np.array_equal(out.numpy(), want)
    g.destroy()
    st.destroy()
