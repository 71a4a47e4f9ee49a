"""The adapters, norms and the gate on tensors that share memory: refused where a result would overwrite what others of its rows are
computed from, right where rows of one buffer merely lie between each other."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def adapters(T, K, N, R=8, L=3, seed=0):
    g = torch.Generator().manual_seed(seed + T)
    r = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()  # noqa: E731
    ids = torch.randint(-1, L, (T,), generator=g, dtype=torch.int32).cuda()
    return r, ids, r(L, R, K), r(L, N, R)


@pytest.mark.parametrize("T", [1, 24, 530])
def test_lora_add_refuses_a_result_over_its_other_inputs(T):
    import applied_ai_amd as A

    r, ids, a, b = adapters(T, 64, 64)
    plan = A.lora_plan(ids, 3)
    buffer = r(2 * T + 4, 64)
    y, x = r(T, 64), buffer[1:T + 1]
    for out in (x, buffer[:T + 1][-T:], buffer[2:T + 2] if T > 1 else x):
        before = buffer.clone()
        with pytest.raises(ValueError):
            A.lora_add(y, x, a, b, plan, out=out)
        assert torch.equal(buffer, before)
    if T > 1:
        with pytest.raises(ValueError):  # shifted by a row against y
            A.lora_add(buffer[:T], r(T, 64), a, b, plan, out=buffer[1:T + 1])
        wide = r(T, 100)
        with pytest.raises(ValueError):  # by some columns
            A.lora_add(wide[:, :64], r(T, 64), a, b, plan, out=wide[:, 30:94])
    if T <= 24:
        with pytest.raises(ValueError):
            A.lora_add(y, x, a, b, plan, out=a.view(-1, 64)[:T])


@pytest.mark.parametrize("T", [1, 24, 530])
def test_rows_of_one_buffer_beside_each_other(T):
    """x, y and the result as columns of one buffer, y in place."""
    import applied_ai_amd as A

    r, ids, a, b = adapters(T, 72, 40, seed=1)
    plan = A.lora_plan(ids, 3)
    buffer = r(T, 72 + 40 + 40)
    x, y, z = buffer[:, :72], buffer[:, 72:112], buffer[:, 112:]
    want = A.lora_add(y.contiguous(), x.contiguous(), a, b, plan)
    assert A.lora_add(y, x, a, b, plan, out=z) is z
    assert torch.equal(z, want)
    assert A.lora_add(y, x, a, b, plan, out=y) is y
    assert torch.equal(y, want)
    go = r(T, 40)
    both = r(T, 144)
    left, right = both[:, :72], both[:, 72:]
    want = A.lora_backward(go, x.contiguous(), a, b, plan, grad_x=left.contiguous())
    got = A.lora_backward(go, x, a, b, plan, grad_x=left, out=right)
    assert got[0] is right and all(torch.equal(p, q) for p, q in zip(got, want))
    got = A.lora_backward(go, x, a, b, plan, grad_x=left, out=left)
    assert got[0] is left and all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("T", [2, 24, 530])
def test_lora_backward_refuses_a_result_over_what_it_is_computed_from(T):
    import applied_ai_amd as A

    r, ids, a, b = adapters(T, 64, 48, seed=2)
    plan = A.lora_plan(ids, 3)
    x, go = r(T, 64), r(T, 48)
    buffer = r(T + 2, 100)
    with pytest.raises(ValueError):
        A.lora_backward(go, x, a, b, plan, grad_x=buffer[:T, :64], out=buffer[1:T + 1, :64])
    with pytest.raises(ValueError):
        A.lora_backward(go, x, a, b, plan, grad_x=buffer[:T, :64], out=buffer[:T, 36:])
    if T <= 24:
        with pytest.raises(ValueError):
            A.lora_backward(go, x, a, b, plan, out=a.view(-1, 64)[:T])
