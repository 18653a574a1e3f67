"""Products queued behind one whose in-launch wait gives up.  Needs a real MI355X (-m gpu)."""
import time

import numpy as np
import pytest

from gpu_helpers import env, pa, reload_switches
from test_gpu_self_exchange import SelfPeriodicPart, _comm

pytestmark = pytest.mark.gpu

import pa_amd._lib as L  # noqa: E402


def test_products_queued_behind_a_time_out_do_not_wait_in_turn():
    """A flag that never comes (PA_TEST_FUSED_SKIP_RAISE=-2: none from the second product on) costs the GPU ONE time-out, however many
    products are queued: each of them sat it out in turn before.  Said once, and the handle goes on as separate launches."""
    limit, queued = 0.5, 12
    with env(PA_IPC_TIMEOUT_S=str(limit), PA_TEST_FUSED_SKIP_RAISE="-2", PA_MUL_FUSED="1", PA_MUL_FUSED_RCCL="1"):
        reload_switches()
        P = SelfPeriodicPart(16)
        ctx = P.ctx
        comm = _comm(ctx)
        x = np.random.default_rng(5).integers(-3, 4, P.n_own).astype(np.float64)
        P.b.upload(np.concatenate([x, np.zeros(P.n_ghost)]))
        L.call("pa_mul5", P.m, comm, P.c.h, P.b.h, 1.0, 0.0)
        ctx.sync()
        assert np.array_equal(P.c.download(), P.expected_integer(x))
        inside0 = ctx.fused_launches()[1]
        t0 = time.perf_counter()
        for _ in range(queued):
            L.call("pa_mul5", P.m, comm, P.c.h, P.b.h, 1.0, 0.0)
        with pytest.raises(L.PAError, match="gave up waiting"):
            ctx.sync()
        took = time.perf_counter() - t0
        assert ctx.fused_launches()[1] - inside0 == queued       # (all were queued before the first gave up)
        assert limit <= took < 3 * limit, took
        ctx.sync()                                               # (said once)
        x = x + 1.0
        P.b.upload(np.concatenate([x, np.zeros(P.n_ghost)]))
        L.call("pa_mul5", P.m, comm, P.c.h, P.b.h, 1.0, 0.0)
        ctx.sync()
        assert np.array_equal(P.c.download(), P.expected_integer(x))
        assert np.array_equal(P.b.download()[P.n_own:], x[P.wrap])
        P.close()
        L.call("pa_comm_destroy", comm)
    reload_switches()
