"""The training step with its optional terms: orthogonalised updates of the Reconstructor's convolutions, an entropy term, top-k statistics."""
import types

import pytest
import torch

from tests import golden_inputs as GI
from tests.test_orthogonalise_gpu import exact, noisy
from warpedganspace_amd import ops
from warpedganspace_amd.gan_load import StyleGAN2Wrapper
from warpedganspace_amd.reconstructor import Reconstructor
from warpedganspace_amd.stylegan2 import Generator
from warpedganspace_amd.support_sets import SupportSets
from warpedganspace_amd.trainer import TrainStep

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


def make(dev, **kw):
    torch.manual_seed(0)
    K, N, B = 16, 4, 4
    G = Generator(32, 512, 8)
    G.load_state_dict(GI.fill_state_dict(G.state_dict(), 932))
    c = GI.support_sets_case(K, N, 512, B, 31, learn_gammas=True)
    S = SupportSets(K, N, 512, learn_gammas=True, gamma=c['gamma'])
    S.load_state_dict(c['sd'])
    R = Reconstructor('ResNet', K)
    p = types.SimpleNamespace(reconstructor_lr=1e-3, support_set_lr=1e-4, min_shift_magnitude=0.25, max_shift_magnitude=0.45, lambda_cls=1.0,
                              lambda_reg=0.25, z_truncation=None, shift_in_w_space=False, **kw)
    return TrainStep(StyleGAN2Wrapper(G, False).to(dev).eval(), S.to(dev).train(), R.to(dev).train(), p, B, dev, seed=1, precision='fp32')


def batch(dev, seed):
    g = torch.Generator().manual_seed(seed)
    return [t.to(dev) for t in (torch.randn(4, 512, generator=g), torch.randint(0, 16, (4,), generator=g), torch.tensor([0.3, -0.4, 0.28, -0.33]))]


def test_steps_with_orthogonalised_updates(dev):
    """Every parameter after each of two steps against the update formulas on the step's own gradients."""
    eng = make(dev, optimizer='muon')
    b = eng.bucket
    convs = [p for p in eng.R.parameters() if p.dim() == 4]
    assert len(convs) == 20 and b.muon_end == sum((p.numel() + 3) // 4 * 4 for p in convs)
    mom = {id(p): torch.zeros(p.numel(), device=dev, dtype=torch.float64) for p in convs}
    m1, m2 = torch.zeros_like(b.flat, dtype=torch.float64), torch.zeros_like(b.flat, dtype=torch.float64)
    for it in range(2):
        before = b.flat.clone()
        eng.step(*batch(dev, it))
        torch.cuda.synchronize()
        g = b.grad.double()
        m1 = m1 + (g - m1) * 0.1
        m2 = 0.999 * m2 + 0.001 * g * g
        for p, off, n in b.segments:
            w0, w1 = before[off:off + n].double(), b.flat[off:off + n].double()
            if id(p) in mom:
                m = mom[id(p)] = 0.95 * mom[id(p)] + g[off:off + n]
                u = (g[off:off + n] + 0.95 * m).view(p.shape[0], -1)
                o = exact(u)
                lr = 1e-3 * 0.2 * max(u.shape) ** 0.5
                err = (w1 - (w0 - lr * o.reshape(-1))).norm()
                # the orthogonalisation's own noise (the update's rounding to fp32 is within it), and the weight's rounding
                allowed = lr * (12 * (noisy(u.float(), [1] * 5) - exact(u.float())).norm() + 2.0 ** -20 * o.norm()) + 1.1 * EPS * w1.norm()
                assert err <= allowed, (it, tuple(p.shape), float(err), float(allowed))
            else:
                lr = 1e-3 if off < b.groups[0][2] else 1e-4
                a, v = m1[off:off + n] / (1 - 0.9 ** (it + 1)), m2[off:off + n] / (1 - 0.999 ** (it + 1))
                want = w0 - lr * a / (v.sqrt() + 1e-8)
                assert float((w1 - want).abs().max()) <= lr * 2e-4 + EPS * float(w1.abs().max())      # (fp32 bias corrections: 1 - 0.999 has 2^-14 steps)
    # the update's length: 0.2 lr per entry, like Adam's
    assert torch.isfinite(b.flat).all()


def test_optimizer_state_round_trip(dev):
    a, b = make(dev, optimizer='muon'), make(dev, optimizer='muon')
    a.step(*batch(dev, 1))
    b.bucket.flat.copy_(a.bucket.flat)
    for x, y in zip(a.R.buffers(), b.R.buffers()):
        y.copy_(x)
    assert b.load_optim_state(a.optim_state())
    assert not make(dev).load_optim_state(a.optim_state())             # another optimizer's moments
    adam = make(dev)
    assert not a.load_optim_state(adam.optim_state())
    old = adam.optim_state()
    del old['optimizer']                                               # written before the key existed: Adam's
    assert adam.load_optim_state(old)
    for e in (a, b):
        e.step(*batch(dev, 2))
    err = (a.bucket.flat - b.bucket.flat).abs().max()
    assert float(err) <= 1e-4, float(err)                              # (atomics in the gradients' sums: not bit for bit)


def test_entropy_term_and_top_accuracy(dev):
    """dlogits, the total loss and the statistics against the formulas in 64 bits on the step's own scores."""
    lam = 0.3
    eng = make(dev, lambda_ent=lam, label_top=3)
    seen = {}
    run = eng._label_terms

    def spy(logits, idx):
        seen.update(logits=logits.detach().clone(), idx=idx.clone(), ce=eng.dlogits.clone(), total=eng.stats[2].clone())
        run(logits, idx)
        seen['after'] = eng.dlogits.clone()
    eng._label_terms = spy
    st = eng.step(*batch(dev, 3)).clone()
    x = seen['logits'].double().requires_grad_(True)
    logp = torch.log_softmax(x, 1)
    ent = -(logp.exp() * logp).sum(1).mean()
    (-lam * ent).backward()
    assert float((seen['after'].double() - seen['ce'].double() - x.grad).abs().max()) <= 64 * EPS * (1 + float(logp.abs().max()))
    assert abs(float(st[2]) - (float(seen['total']) - lam * float(ent))) <= 16 * EPS * (1 + abs(float(st[2])))
    top = (x.topk(3, 1).indices == seen['idx'][:, None]).any(1).double().mean()
    out = eng.pop_stats()
    assert abs(out['entropy'] - float(ent)) <= 64 * EPS * (1 + float(ent)) and out['top3_accuracy'] == float(top)
    assert set(make(dev).pop_stats()) == {'accuracy', 'classification_loss', 'regression_loss', 'total_loss'}


def test_the_operators_together(dev):
    """A classifier trained by them alone: scores, log-probabilities with entropy, their gradient, orthogonalised updates; the gradients against
    those of the same loss in 64 bits, the weights against the update formula."""
    gen = torch.Generator(device=dev).manual_seed(0)
    x = torch.randn(64, 96, generator=gen, device=dev)
    y = torch.randint(0, 40, (64,), generator=gen, device=dev)
    y[::7] = -100
    w = (0.1 * torch.randn(40, 96, generator=gen, device=dev)).requires_grad_(True)
    m = torch.zeros(40, 96, device=dev)
    for _ in range(3):
        r = ops.label_logprobs(x @ w.t(), y, top=2)
        loss = -r.logp.mean() - 0.05 * r.entropy.mean() - 0.01 * r.top_logp.mean()
        grad, = torch.autograd.grad(loss, w)
        w64 = w.detach().double().requires_grad_(True)
        lp = torch.log_softmax(x.double() @ w64.t(), 1)
        given = torch.where(y >= 0, lp.gather(1, y.clamp(min=0)[:, None])[:, 0], torch.zeros_like(lp[:, 0]))
        want, = torch.autograd.grad(-given.mean() + 0.05 * (lp.exp() * lp).sum(1).mean() - 0.01 * lp.topk(2, 1).values.mean(), w64)
        # fp32 products of 96 and 64 terms and a log-softmax of 40: some 200 roundings of the terms' size
        assert float((grad.double() - want).abs().max()) <= 256 * EPS * float((x.abs().sum(0).max() / 64).double())
        old, m0 = w.detach().double().clone(), m.double()
        with torch.no_grad():
            ops.muon_step([w], [grad], [m], 0.02)
        mm = 0.95 * m0 + grad.double()
        u = grad.double() + 0.95 * mm
        noise = (noisy(u.float(), [1] * 5) - exact(u.float())).norm()
        err = (w.detach().double() - (old - 0.02 * exact(u))).norm()
        assert float(err) <= 0.02 * float(12 * noise + 2.0 ** -20 * exact(u).norm()) + 1.1 * EPS * float(old.norm())
