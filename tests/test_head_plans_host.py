"""Plans of the classifier head's loss, without a GPU: scratch sizes, what is refused, documentation that compiles."""
import ctypes

import pytest

import cudnntest_b200 as cb


def _bytes(plan, grad):
    return cb.lib().wino_xent_workspace_bytes(ctypes.byref(plan.desc), grad)


@pytest.mark.parametrize("n,d,v,kw", [
    (677, 9184, 1383, dict(label_smoothing=0.1, scratch_limit=16 << 20)),         # dz counts against the limit with gradients alone
    (1457, 1, 7119, dict()),                                                      # plain kernels without gradients alone
    (14201, 1, 393, dict(scratch_limit=16 << 20, bias=True)),
    (58, 5, 4892, dict(scratch_limit=1, dtype="fp32x3")),
    (64, 4096, 1000, dict()), (1, 1, 1, dict()), (0, 8, 8, dict()), (4096, 1024, 32000, dict(dtype="fp32x3")),
])
def test_a_plan_with_gradients_has_room_for_forward(n, d, v, kw):
    """`forward` may be called on it: its scratch is at least that of either call."""
    plan = cb.LinearXent(n, d, v, device="meta", **kw)
    need = max(_bytes(plan, 0), _bytes(plan, 1))
    assert plan.ws_bytes >= need and plan.workspace.numel() >= need
    alone = cb.LinearXent(n, d, v, device="meta", grad=False, **kw)
    assert alone.ws_bytes == _bytes(alone, 0)
