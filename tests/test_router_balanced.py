"""Router with the balance loss and counts against its definition in 64 bits.

Tolerances: probabilities come from one fp32 exponential (argument below ~30: 30 * 2^-23
relative, and 2^-21 of the hardware exponential with its scaled argument), a sum of E terms
(E / 32 + 5 roundings of 2^-24) and a division: ``_P`` relative. The mean of p over tokens adds one rounding per
token that a warp meets (T / (8 * blocks)) before the 64-bit sums.
"""
import math

import pytest
import torch

_P = 2.0**-20 + 32 * 2.0**-23
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _inputs(T, E, dtype, seed, strided=False):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, E, generator=g) * 1.5).bfloat16().to(DT[dtype])  # bf16 values: ties are exact
    if strided:
        wide = torch.full((T, E + 3), math.nan, dtype=DT[dtype])
        wide[:, 1:1 + E] = x
        return wide.cuda()[:, 1:1 + E].requires_grad_(), g
    return x.cuda().requires_grad_(), g


def _check(x, k, renorm, bias, valid, dw, up):
    from spec_ep.ops.router import router_topk_balanced, router_topk_balanced_reference

    T, E = x.shape
    w, e, loss, counts = router_topk_balanced(x, k, renorm, bias, valid)
    xr = x.detach().double().requires_grad_()
    wr, er, lr, cr = router_topk_balanced_reference(xr, k, renorm, None if bias is None else bias.double(), valid)
    assert torch.equal(e, er) and e.dtype == torch.int32
    assert torch.equal(counts, cr) and counts.dtype == torch.int32
    assert ((w.double() - wr).abs() <= wr * 4 * _P + 1e-30).all()
    assert abs(loss.item() - lr.item()) <= lr.item() * (2 * _P + T * 2.0**-24 / 8)
    (g,) = torch.autograd.grad([w, loss], x, [dw, up])
    (gr,) = torch.autograd.grad([wr, lr], xr, [dw.double(), up.double()])
    assert g.dtype == x.dtype and g.shape == x.shape
    # dx = p (g - sum p g): errors of p times the largest term, and one rounding
    p = torch.softmax(xr, 1).detach()
    S = wr.new_tensor(1.0) if not renorm else p.gather(1, er.long()).sum(1, keepdim=True).detach()
    n = max(int(valid.sum()), 1) if valid is not None else max(T, 1)
    big = (dw.abs().amax(1, keepdim=True).double() * 2 / S + up.abs().double() * E / n)
    tol = gr.abs() * torch.finfo(x.dtype).eps / 2 + p * big * 16 * _P
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    assert ((g.double() - gr).abs() <= tol + tiny).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (7, 13, 13), (300, 128, 8), (65, 60, 4), (33, 160, 6),
                                   (50, 257, 10), (20, 512, 32), (5000, 64, 6)])
def test_balanced_router(T, E, k, dtype):
    x, g = _inputs(T, E, dtype, T + E, strided=T == 65)
    dw = torch.randn(T, k, generator=g).cuda()
    up = torch.tensor(0.7, device="cuda")
    valid = (torch.rand(T, generator=g) < 0.6).cuda()
    for renorm in (True, False):
        _check(x, k, renorm, None, None, dw, up)
        _check(x, k, renorm, None, valid, dw, up)


@pytest.mark.gpu
def test_selection_bias_leaves_the_weights_alone():
    """A bias far above the probabilities' errors decides the selection."""
    T, E, k = 200, 32, 4
    x, g = _inputs(T, E, "fp32", 1)
    bias = (4.0 * torch.randperm(E, generator=g).float()).cuda()
    _check(x, k, True, bias, None, torch.randn(T, k, generator=g).cuda(), torch.tensor(1.0, device="cuda"))


@pytest.mark.gpu
def test_agrees_with_router_topk():
    from spec_ep.ops.router import router_topk, router_topk_balanced

    x, _ = _inputs(512, 128, "fp32", 2)
    x = (x.detach() + torch.rand(512, 128, device="cuda") * 2.0**-3)  # no ties
    w, e = router_topk(x, 8)
    w2, e2, _, counts = router_topk_balanced(x, 8)
    assert torch.equal(e, e2) and (w - w2).abs().max().item() < 1e-6
    assert torch.equal(counts.long(), torch.bincount(e.reshape(-1), minlength=128))


@pytest.mark.gpu
def test_uniform_router_has_loss_one_and_ties_go_to_the_lowest_index():
    from spec_ep.ops.router import router_topk_balanced

    x = torch.zeros(64, 16, device="cuda", requires_grad=True)
    with torch.no_grad():
        x[1] = -0.0  # equal to +0
        x[2, ::2] = -0.0
    w, e, loss, counts = router_topk_balanced(x, 3)
    assert torch.equal(e.cpu(), torch.arange(3, dtype=torch.int32).expand(64, 3))
    assert (w - 1 / 3).abs().max().item() < 1e-6
    assert counts.tolist() == [64] * 3 + [0] * 13
    assert abs(loss.item() - 1.0) < 1e-5  # any counts against uniform probabilities


@pytest.mark.gpu
def test_masked_experts_and_extreme_rows():
    """-inf and lowest-value logits, fewer finite ones than k, and NaN rows: indices stay
    distinct and inside the range."""
    from spec_ep.ops.router import router_topk_balanced

    E, k = 40, 6
    x = torch.randn(6, E, device="cuda")
    x[0, 2:] = -math.inf
    x[1, 5:] = torch.finfo(torch.float32).min
    x[2] = math.nan
    x[3, 7] = math.nan
    x[4, 3] = -math.nan
    x[5] = -math.inf
    w, e, loss, counts = router_topk_balanced(x, k)
    for row in e.tolist():
        assert len(set(row)) == k and all(0 <= i < E for i in row)
    assert sorted(e[0].tolist()[:2]) == [0, 1] and e[0].tolist()[2:] == [2, 3, 4, 5]
    assert w[0, 2:].abs().max().item() == 0 and w[:2].isfinite().all()
    assert e[3, 0].item() == 7
    assert counts.sum().item() == 6 * k
    # NaN rows out of the mask do not reach the loss
    valid = torch.tensor([1, 1, 0, 0, 0, 0], device="cuda").bool()
    x.requires_grad_()
    w, e, loss, counts = router_topk_balanced(x, k, valid=valid)
    assert loss.isfinite() and counts.sum().item() == 2 * k
    (g,) = torch.autograd.grad(loss, x)
    assert g[:2].isfinite().all()


@pytest.mark.gpu
def test_only_one_of_the_outputs_used_and_empty_batches():
    from spec_ep.ops.router import router_topk_balanced

    x, g = _inputs(100, 24, "fp32", 3)
    dw = torch.randn(100, 4, generator=g).cuda()
    w, e, loss, _ = router_topk_balanced(x, 4)
    (both,) = torch.autograd.grad([w, loss], x, [dw, torch.tensor(2.0, device="cuda")], retain_graph=True)
    (a,) = torch.autograd.grad(w, x, dw, retain_graph=True)
    (b,) = torch.autograd.grad(loss, x, torch.tensor(2.0, device="cuda"))
    assert (a + b - both).abs().max().item() < 1e-6 * both.abs().max().item() + 1e-7
    none = torch.zeros(100, dtype=torch.bool, device="cuda")
    w, e, loss, counts = router_topk_balanced(x, 4, valid=none)
    (gz,) = torch.autograd.grad(loss, x)
    assert loss.item() == 0 and not counts.any() and not gz.any()
    y = torch.zeros(0, 24, device="cuda", requires_grad=True)
    w, e, loss, counts = router_topk_balanced(y, 4)
    (gz,) = torch.autograd.grad([w, loss], y, [torch.zeros(0, 4, device="cuda"), torch.tensor(1.0, device="cuda")])
    assert loss.item() == 0 and gz.shape == (0, 24) and e.shape == (0, 4)


@pytest.mark.gpu
def test_balance_gradient_against_differences():
    """h = 2^-5: rounding of a loss near 1 gives 2^-23 / h < 4e-6, h^2 / 6 times the third
    derivative (below 1 along a direction of size 1) 2e-4. Distinct logits keep the choice."""
    from spec_ep.ops.router import router_topk_balanced

    T, E, k, h = 16, 12, 3, 2.0**-5
    x = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(i)) for i in range(T)]).float().cuda() / 4
    x.requires_grad_()
    cw = torch.randn(T, k, generator=torch.Generator().manual_seed(1)).cuda()

    def f(v):
        w, e, loss, _ = router_topk_balanced(v, k)
        return (w * cw).sum() / T + loss

    (g,) = torch.autograd.grad(f(x), x)
    gen = torch.Generator().manual_seed(2)
    for _ in range(4):
        d = torch.rand(T, E, generator=gen).cuda() * 2 - 1
        with torch.no_grad():
            diff = (f(x + h * d).double() - f(x - h * d).double()) / (2 * h)
        assert abs(diff.item() - (g.double() * d).sum().item()) < 1e-3


@pytest.mark.gpu
def test_same_bits_on_every_run_another_stream_and_in_graphs():
    from spec_ep.ops.router import router_topk_balanced

    xa, g = _inputs(3000, 128, "bf16", 4)
    xb, _ = _inputs(3000, 128, "bf16", 5)
    dw, up = torch.randn(3000, 8, generator=g).cuda(), torch.tensor(0.3, device="cuda")

    def one(x):
        w, e, loss, counts = router_topk_balanced(x, 8)
        (gx,) = torch.autograd.grad([w, loss], x, [dw, up])
        return w, e, loss, counts, gx

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = one(xa)
        one(xb)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, one(xa)):
        assert torch.equal(a, b)
    outs, graphs = [], []
    for x in (xa, xb):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(one(x))
        graphs.append(gr)
    for _ in range(2):
        with torch.no_grad():
            xa.copy_(xa.roll(1, 1))
            xb.mul_(0.5)
        for gr in graphs:
            gr.replay()
        for x, o in zip((xa, xb), outs):
            for a, b in zip(o, one(x)):
                assert torch.equal(a, b)


def test_router_refusals():
    from spec_ep.ops.router import router_topk_balanced

    x = torch.zeros(4, 8)

    def refused(*a, match, **kw):
        with pytest.raises((RuntimeError, ValueError), match=match):
            router_topk_balanced(*a, **kw)

    refused(x, 2, match="CUDA")
    refused(x[0], 2, match=r"\[T, E\]")
    refused(x, 0, match="k must be")
    refused(x, 9, match="k must be")
    refused(torch.zeros(4, 600), 2, match="experts")
    refused(x.double(), 2, match="bf16, fp16 or fp32")
    refused(torch.zeros(8, 4).t(), 2, match="unit stride")
    refused(x, 2, valid=torch.ones(3, dtype=torch.bool), match="valid")
    refused(x, 2, valid=torch.ones(4), match="valid")
    refused(x, 2, bias=torch.zeros(7), match="bias")
    refused(x, 2, bias=torch.zeros(8).double(), match="bias")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,E", [(1, 1), (40, 13), (600, 128), (90, 512)])
def test_one_choice_with_weight_one_gets_no_gradient_through_it(T, E, dtype):
    """k = 1, renormalised: the weight is 1 whatever the logits are, so the gradient is that
    of the balance loss alone, to the bit, however small it is beside the weights'."""
    from spec_ep.ops.router import router_topk_balanced

    x, g = _inputs(T, E, dtype, T + E)
    dw, up = 100.0 * torch.randn(T, 1, generator=g).cuda(), torch.tensor(0.01, device="cuda")
    w, _, loss, _ = router_topk_balanced(x, 1)
    assert (w == 1.0).all()
    (both,) = torch.autograd.grad([w, loss], x, [dw, up], retain_graph=True)
    (alone,) = torch.autograd.grad(loss, x, up)
    assert torch.equal(both, alone)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [4.0, 12.0])
def test_gradient_of_nearly_certain_choices(d):
    """Two choices whose logits lie d apart: dx_0 = w_0 w_1 (dw_0 - dw_1) = -dx_1, small
    beside dw. Relative errors: d 2^-23 of the exponential's argument (the product's rounding
    and the constant's, each d 2^-24), 2 * 2^-23 of the exponential, and below 20 roundings
    of 2^-24 or divisions of 2^-23 from the sums, weights and products."""
    from spec_ep.ops.router import router_topk_balanced

    T = 256
    g = torch.Generator().manual_seed(int(d))
    x = torch.tensor([0.0, -d]).repeat(T, 1).cuda().requires_grad_()
    dw = torch.randn(T, 2, generator=g).cuda()
    w, _, _, _ = router_topk_balanced(x, 2)
    (gx,) = torch.autograd.grad(w, x, dw)
    w1 = 1.0 / (1.0 + math.exp(d))
    want = w1 * (1.0 - w1) * (dw[:, 0] - dw[:, 1]).double()
    for got, sign in ((gx[:, 0], 1.0), (gx[:, 1], -1.0)):
        assert ((got.double() - sign * want).abs() <= want.abs() * (d + 22) * 2.0**-23).all()
