"""NaN scores of either sign come before every number, the lowest index first."""
import pytest
import torch


def _nan(sign, dtype):
    """NaN with the given sign bit, as the host's 0/0 (negative) or a literal has it."""
    bits = {torch.float32: (0x7FC00000, torch.int32), torch.bfloat16: (0x7FC0, torch.int16),
            torch.float16: (0x7E00, torch.int16)}[dtype]
    v = torch.tensor([bits[0]], dtype=torch.int64)
    if sign < 0:
        v |= torch.tensor([-(1 << 31) if dtype == torch.float32 else -(1 << 15)])
    return v.to(bits[1]).view(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("E", [40, 128, 512])
def test_nan_of_either_sign_is_chosen_first(E, dtype, bias):
    from spec_ep.ops.router import router_topk_balanced

    for seed in range(3):
        x = torch.randn(5, E, generator=torch.Generator().manual_seed(seed)).to(dtype)
        neg, pos = _nan(-1, dtype), _nan(1, dtype)
        assert neg.isnan() and pos.isnan() and torch.signbit(neg) and not torch.signbit(pos)
        x[0, 3] = neg
        x[1, 3] = pos
        x[2, 30], x[2, 17] = neg, pos
        x[3, 30], x[3, 17] = pos, neg
        x[4, :] = neg
        x = x.cuda()
        b = torch.zeros(E, device="cuda") if bias else None
        if bias:  # a NaN logit makes all of its row's probabilities NaN: the bias's NaN instead
            x = torch.where(x.isnan(), torch.zeros_like(x), x)
            b[17], b[30] = neg.float().item(), neg.float().item()
            b[17:18].view(torch.int32).fill_(-0x00400000)
            _, e, _, _ = router_topk_balanced(x, 4, bias=b)
            assert (e[:, 0] == 17).all() and (e[:, 1] == 30).all()
            continue
        _, e, _, _ = router_topk_balanced(x, 4)
        assert e[:2, 0].tolist() == [3, 3]
        assert e[2:4, :2].tolist() == [[17, 30], [17, 30]]
        assert e[4].tolist() == [0, 1, 2, 3]
