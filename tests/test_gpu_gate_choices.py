"""The router's gate with more choices than 32 of up to 256 experts: forms of one wave to a row."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k", [(9, 60, 40), (5, 64, 64), (3, 33, 33), (7, 200, 50), (6, 256, 33), (4, 65, 64)])
def test_many_choices(T, E, k, score, renormalize):
    from test_gpu_gate import test_forward_and_backward as check

    check(T, E, k, score, renormalize)
