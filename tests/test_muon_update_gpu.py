"""The momentum step as a PyTorch user meets it: graphs that hold its tensors, tensors that overlap, gradients that are made anew."""
import pytest
import torch

from tests.test_orthogonalise_gpu import check
from warpedganspace_amd import _lib as L
from warpedganspace_amd import ops

pytestmark = pytest.mark.gpu


def test_a_graph_that_saved_a_weight_before_the_step_is_refused(dev):
    w = torch.randn(12, 20, device=dev, requires_grad=True)
    g, m = torch.randn(12, 20, device=dev), torch.zeros(12, 20, device=dev)
    before = w._version, m._version, g._version
    loss, product = w.square().sum(), (m * w).sum()
    ops.muon_step([w], [g], [m], 0.1)
    assert w._version > before[0] and m._version > before[1] and g._version == before[2]
    for late in (loss, product):
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            late.backward()
    w.square().sum().backward()                # of the new weight
    assert torch.equal(w.grad, 2 * w.detach())
    plan = ops.MuonUpdate([w], [g], [m])
    loss = w.square().sum()
    plan.step(0.1)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()
    with torch.inference_mode():               # tensors without a counter are stepped as ever
        t = [torch.randn(4, 6, device=dev) for _ in range(2)] + [torch.zeros(4, 6, device=dev)]
        old = t[0].clone()
        ops.muon_step([t[0]], [t[1]], [t[2]], 0.1)
        assert not torch.equal(t[0], old)


@pytest.mark.parametrize('order', [1, -1])
def test_a_large_matrix_beside_a_long_batch_of_short_ones(dev, order):
    """Together they would pass the largest grid of the norm's launch."""
    big, short = torch.randn(2048, 2048, device=dev), torch.randn(70000, 17, 17, device=dev)
    got = ops.orthogonalise([big, short][::order])[::order]
    assert torch.equal(got[0], ops.orthogonalise(big))
    check(got[1][::997], short[::997])         # (in the launches of the large one some take another path than by themselves)


@pytest.mark.parametrize('order', [1, -1])
def test_a_large_matrix_beside_a_long_batch_of_single_entries(dev, order):
    big, small = torch.randn(2048, 2048, device=dev), torch.randn(70000, 1, 1, device=dev)
    got = ops.orthogonalise([big, small][::order])[::order]
    assert torch.equal(got[0], ops.orthogonalise(big))
    a, b, c = ops.NS_COEFFICIENTS           # (the smallest of 70000 normal samples is some 1e-5: eps counts a little)
    y = small.double() / (small.double().abs() + 1e-7)
    for _ in range(5):
        y = y * (a + b * y ** 2 + c * y ** 4)
    # a step multiplies a relative error by at most |1 + 2 (b A + 2 c A^2) / (a + b A + c A^2)| < 8 for y of 0.5 .. 1.2; pairs of 22 bits
    assert float((got[1].double() - y).abs().max()) < 2e-4


def test_a_gradient_that_was_made_anew_is_not_taken_for_the_old_one(dev):
    w = torch.randn(6, 9, device=dev, requires_grad=True)
    x = torch.randn(9, 4, device=dev)
    m = torch.zeros(6, 9, device=dev)
    (w @ x).sum().backward()
    plan = ops.MuonUpdate([w], [w.grad], [m])
    plan.step(0.1)
    w.grad.zero_()                             # zero_grad(set_to_none=False): the same tensor
    (w @ x).sum().backward()
    plan.step(0.1)
    old = w.detach().clone()
    for again in (False, True):
        w.grad = None                          # zero_grad(): the next backward makes a new tensor
        if again:
            (w @ x).sum().backward()
        with pytest.raises(L.WgsError, match='another tensor'):
            plan.step(0.1)
    assert torch.equal(w, old)
    ops.MuonUpdate([w], [w.grad], [m]).step(0.1)
    g = torch.randn(6, 9, device=dev)          # a gradient of one's own: .grad does not matter
    plan = ops.MuonUpdate([w], [g], [m])
    w.grad = None
    plan.step(0.1)


def test_captured_steps_of_few_rows_among_others(dev):
    """Replays read the buffers' current contents, with eager work in between; two graphs do not share a workspace."""
    shapes = [(5, 70), (40, 90), (900, 16), (1, 1)]

    def state(seed):
        gen = torch.Generator(device=dev).manual_seed(seed)
        return [[torch.randn(s, generator=gen, device=dev) for s in shapes] for _ in range(3)]
    cap, ref = [state(1), state(2)], [state(1), state(2)]
    ops.muon_step(*state(3), 0.1)
    torch.cuda.synchronize()
    graphs = []
    for s in cap:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.muon_step(*s, 0.1, weight_decay=0.1)
        graphs.append(g)
    for k in range(3):
        fresh = state(10 + k)[1]
        for i in (0, 1):
            for a, b, new in zip(cap[i][1], ref[i][1], fresh):
                a.copy_(new * (i + 1))
                b.copy_(new * (i + 1))
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            ops.muon_step(*ref[i], 0.1, weight_decay=0.1)
            for a, b in zip(cap[i][0] + cap[i][2], ref[i][0] + ref[i][2]):
                assert torch.equal(a, b), (k, i)
