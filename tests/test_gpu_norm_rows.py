"""The gradients of the norms around a block where rows have no columns, and where a workgroup adds up many rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("T", [1, 300])
@pytest.mark.parametrize("weights", [BF, F32])
def test_rows_without_columns(T, weights):
    """A gate per row is the only argument with elements: its gradient is an empty sum, zero."""
    import applied_ai_amd as A
    from applied_ai_amd import ops

    y, gate = torch.empty(T, 0, dtype=BF).cuda(), torch.ones(T, 1, dtype=weights).cuda()
    h, z = A.block_norm(y, y, None, gate)
    assert h.shape == (T, 0) and z is None
    got = A.block_norm_backward(y, None, y, y, None, gate)
    assert got[3].shape == (T, 1) and got[3].dtype == weights and not got[3].any()
    old = torch.full((T + 1, 1), float("nan"), dtype=weights).cuda()
    kind = 2 if weights == F32 else 0
    rc = A._lib.lib().moe_gg_block_norm_backward(None, 0, None, 0, None, 0, None, 0, None, gate.data_ptr(), 2, None, 1.0, 1.0, 1e-6, None, None, None,
                                                 old.data_ptr(), None, T, 0, 0, 0, kind, None, 0, ops._stream_ptr(old.device))
    assert rc == 0 and not old[:T].any() and bool(old[T].isnan().all())
