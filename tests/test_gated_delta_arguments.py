"""What the gated delta rule says of operands that have too few or too many dimensions, before it looks at a device."""
import pytest

torch = pytest.importorskip("torch")


def _operands(*v):
    q = torch.zeros(2, 3, 1, 64, dtype=torch.bfloat16)
    return q, q, torch.zeros(v, dtype=torch.bfloat16), torch.zeros(2, 3, 2), torch.zeros(2, 3, 2)


@pytest.mark.parametrize("v", [(2, 3, 128), (2, 3), (6,), (2, 3, 2, 64, 1)])
def test_values_of_other_dimensions(v):
    from rwkv_next_amd.kernels import gated_delta, gated_delta_pool_, gated_delta_pool_op
    with pytest.raises(ValueError, match=r"v \(B, T, Hv, V\)"):
        gated_delta(*_operands(*v))
    with pytest.raises(ValueError, match=r"v \(B, T, Hv, V\)"):
        gated_delta_pool_(*_operands(*v), torch.zeros(4, 2, 64, 64), torch.tensor([0, 1]))
    with pytest.raises(ValueError, match=r"v \(B, T, Hv, V\)"):
        gated_delta_pool_op(*_operands(*v), torch.zeros(4, 2, 64, 64), torch.tensor([0, 1]), None, None, None, None, False, True, True,
                            None, None, -1)


def test_queries_of_other_dimensions():
    from rwkv_next_amd.kernels import gated_delta, gated_delta_pool_
    q, k, v, g, beta = _operands(2, 3, 2, 64)
    with pytest.raises(ValueError, match=r"q, k .*\(B, T, Hk, K\)"):
        gated_delta(q.flatten(2), k, v, g, beta)
    with pytest.raises(ValueError, match=r"q, k .*\(B, T, Hk, K\)"):
        gated_delta_pool_(q.flatten(2), k, v, g, beta, torch.zeros(4, 2, 64, 64), torch.tensor([0, 1]))
