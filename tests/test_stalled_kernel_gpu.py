"""A kernel of an asynchronous call whose bounded wait gave up: synchronize says so, once, and later calls do not.

The wait runs out after a few polls of a barrier that nothing arrives at; the kernel ends by itself."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_synchronize_reports_a_wait_that_gave_up():
    from vokra_b200 import _lib, ops, synth
    from vokra_b200._lib import VkbError
    L = _lib.load()
    ctx = ops.Context(0)
    ctx.synchronize()
    for polls in (1, 1000):
        assert L.vkb_context_selftest_stalled_kernel(ctx.h, polls) == 0
        with pytest.raises(VkbError, match="gave up") as e:
            ctx.synchronize()
        assert e.value.code == _lib.ERROR_OTHER
        ctx.synchronize()
    # and the next call that looks at the flag has nothing to report
    n, k, m = 128, 256, 2
    wq = synth.quantize(synth.Q8_0, np.full(n * k, 0.5, np.float32))
    out = np.zeros((m, n), np.float32)
    ops.gemm_q_f32(ctx, m, n, k, np.ones((m, k), np.float32), wq, synth.Q8_0, None, out)
    assert np.allclose(out, 0.5 * k, rtol=1e-2)
    assert L.vkb_context_selftest_stalled_kernel(ctx.h, 0) == _lib.ERROR_INVALID_ARGUMENT
    assert L.vkb_context_selftest_stalled_kernel(None, 1) == _lib.ERROR_INVALID_ARGUMENT
