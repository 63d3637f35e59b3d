"""Backward passes of the losses from two threads, and captured apart from their forward."""
import threading

import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("i", [0, 1, 2])
def test_two_threads_differentiate_one_kept_graph(i):
    from test_vocab_losses import _logits, _three

    z, _ = _logits(333, 5003, "bf16", False, 1)
    up = torch.tensor(0.3, device="cuda")
    for _ in range(5):
        loss = _three(z, i)
        got = [None, None]

        def run(k):
            got[k] = torch.autograd.grad(loss, z, up, retain_graph=True)[0]

        threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert got[0].data_ptr() != got[1].data_ptr()
        # one of them scales the gradient formed in the forward (two roundings to bf16, 2^-8
        # each), the other forms it from the scaled factor (one)
        assert ((got[0] - got[1]).abs().float() <= 3 * 2.0**-8 * got[0].abs().float() + 1e-30).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("i", [0, 1, 2])
def test_backward_captured_apart_from_its_forward(i, dtype):
    """An eager forward, its backward captured and replayed: every replay gives the same
    gradient, and the forward's own buffers are left alone."""
    from test_vocab_losses import _logits, _three

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z, _ = _logits(33, 1003, dtype, False, 1)
        up = torch.tensor(4.0, device="cuda")  # a power of two: exact where it is applied last
        want = torch.autograd.grad(_three(z, i), z, up)[0]
        loss = _three(z, i)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        (g,) = torch.autograd.grad(loss, z, up, retain_graph=True)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(g, want)
    with torch.cuda.stream(side):  # and the kept graph still gives it
        (again,) = torch.autograd.grad(loss, z, up)
    torch.cuda.synchronize()
    assert torch.equal(again, want)
