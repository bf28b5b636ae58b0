"""GPU, world_size 2 on one device: the data-parallel branches of TrainStep (lib/trainer.py:162-166 is nn.DataParallel in the reference; here one
process per rank) over gloo, which is given host tensors only — by the engine itself (trainer.all_reduce / broadcast) and by these tests.

Each rank runs the same shard through a world = 1 engine, then through a world = 2 engine built from identical weights: replicas start from rank 0's
parameters, the all-reduced gradient bucket is the sum of the ranks' world = 1 gradients, the parameters after the step are Adam's on the averaged
gradient and the same on both ranks, statistics are averaged, the samplers differ; and Trainer.train over two ranks with a TensorBoard writer on rank
0 alone.  Tolerances: the weight gradients' split sums are atomic, so two runs differ by reordered fp32 sums (2e-5 of the largest entry); one Adam
step moves an entry by 1e-4, its error is that of the gradient's relative one (2e-6)."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from tests.test_distributed_gpu import _build, _FakeWriter, _free_port

pytestmark = pytest.mark.gpu


def _host_only():
    """Collectives of device tensors raise."""
    for name in ('all_reduce', 'broadcast'):
        def checked(t, *a, _run=getattr(dist, name), **k):
            assert not t.is_cuda, 'a device tensor was handed to gloo'
            return _run(t, *a, **k)
        setattr(dist, name, checked)


def _start(rank, world, port):
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port), HSA_ENABLE_IPC_MODE_LEGACY='0')
    torch.cuda.set_device(0)
    dist.init_process_group('gloo', rank=rank, world_size=world)
    _host_only()
    return torch.device('cuda', 0)


def _sum(t):
    h = t.cpu()
    dist.all_reduce(h)
    return h.to(t.device)


def _first(t):
    h = t.cpu()
    dist.broadcast(h, 0)
    return h.to(t.device)


def _step_worker(rank, world, port, q):
    try:
        dev = _start(rank, world, port)
        B = 2
        e1, c = _build(dev, 11, 1, 0, B)
        sl = slice(rank * B, (rank + 1) * B)
        z, idx = c['z'][sl].to(dev), c['idx'][sl].to(dev)
        mag = torch.tensor([0.3, -0.4, 0.35, 0.28])[sl].to(dev)
        p0 = e1.bucket.flat.clone()

        def warm(e):     # the generator's lazy weight caches, then the two-stream schedule of a steady-state step
            with torch.no_grad():
                e.G(z)
            torch.cuda.synchronize()
            e.steps_done = 1
        warm(e1)
        st1 = e1.step(z, idx, mag).clone()
        g_local = e1.bucket.grad.clone()
        e2, _ = _build(dev, 11 + rank, world, rank, B)          # rank 1 starts from other reconstructor weights
        start = bool(torch.equal(e2.bucket.flat, p0))
        e2.comm_events = []
        warm(e2)
        e2.step(z, idx, mag)
        torch.cuda.synchronize()
        expect = _sum(g_local)
        err_g = float((e2.bucket.grad - expect).abs().max()) / float(expect.abs().max())
        g = (expect / world).double()                           # Adam's first step: m = (1 - b1) g, v = (1 - b2) g^2, bias-corrected
        upd = torch.zeros_like(g)
        for lr, a, b in e2.bucket.groups:
            upd[a:b] = lr * g[a:b] / (g[a:b].abs() + 1e-8)
        big = g.abs() > 1e-3 * g.abs().max()
        err_p = float((e2.bucket.flat.double() - (p0.double() - upd))[big].abs().max())
        same = bool(torch.equal(e2.bucket.flat, _first(e2.bucket.flat)))
        err_s = abs(e2.pop_stats()['total_loss'] - float(_sum(st1[2:3])) / world)
        zs, _, _ = e2.sample()
        first = _first(zs)
        differs = rank == 0 or not torch.equal(zs, first)
        q.put((rank, start, err_g, err_p, same, err_s, differs, len(e2.comm_events), None))
        dist.barrier()
        dist.destroy_process_group()
    except Exception:  # noqa: BLE001
        import traceback
        q.put((rank,) + (None,) * 7 + (traceback.format_exc(),))
        raise


def _run(worker, *args):
    world, port = 2, _free_port()
    ctx = mp.get_context('spawn')
    torch.cuda.empty_cache()                 # the two ranks share this device with the test process's cached blocks
    q = ctx.Queue()
    procs = [ctx.Process(target=worker, args=(r, world, port) + args + (q,)) for r in range(world)]
    for p in procs:
        p.start()
    try:
        res = sorted((q.get(timeout=100) for _ in range(world)), key=lambda r: r[0])
    finally:
        for p in procs:
            p.join(10)
            if p.is_alive():
                p.kill()
    for r in res:
        assert r[-1] is None, r[-1]
    assert all(p.exitcode == 0 for p in procs)
    return res


def test_trainstep_world2_matches_the_sum_of_the_ranks_gradients(dev):
    for rank, start, err_g, err_p, same, err_s, differs, n_ev, _ in _run(_step_worker):
        assert start, "replicas start from rank 0's parameters"
        assert err_g < 2e-5 and err_p < 2e-6, (err_g, err_p)
        assert same and differs and n_ev == 1
        assert err_s < 1e-5


def _train_worker(rank, world, port, root, q):
    try:
        import types
        from warpedganspace_amd.gan_load import build_stylegan2
        from warpedganspace_amd.reconstructor import Reconstructor
        from warpedganspace_amd.support_sets import SupportSets
        from warpedganspace_amd.trainer import Trainer
        _start(rank, world, port)
        p = types.SimpleNamespace(reconstructor_lr=1e-4, support_set_lr=1e-4, min_shift_magnitude=0.25, max_shift_magnitude=0.45, lambda_cls=1.0,
                                  lambda_reg=0.25, z_truncation=None, shift_in_w_space=False, tensorboard=False, log_freq=3, ckp_freq=1000, max_iter=6,
                                  batch_size=4, seed=3, precision='fp32', lambda_ent=0.1, label_top=2, optimizer='muon')
        torch.manual_seed(0)
        G = build_stylegan2(None, resolution=32)
        S = SupportSets(8, 4, 512, learn_alphas=False, learn_gammas=True, gamma=1.0 / 512)
        R = Reconstructor('ResNet', 8)
        tr = Trainer(params=p, exp_dir='exp', use_cuda=True, root=os.path.join(root, 'r%d' % rank))
        if rank == 0:
            tr.tb_writer = _FakeWriter()
        eng = tr.train(G, S, R)
        same = bool(torch.equal(eng.bucket.flat, _first(eng.bucket.flat)))
        q.put((rank, tr.tb_active, len(tr.tb_writer.rows) if rank == 0 else 0, same, eng.steps_done, None))
        dist.barrier()
        dist.destroy_process_group()
    except Exception:  # noqa: BLE001
        import traceback
        q.put((rank, None, None, None, None, traceback.format_exc()))
        raise


def test_trainer_loop_with_a_writer_on_rank_0_alone(dev, tmp_path):
    """Both ranks read the statistics (an all-reduce) in every iteration; six of them an iteration with the optional terms."""
    res = _run(_train_worker, str(tmp_path))
    assert [r[1] for r in res] == [True, True] and res[0][2] == 6 * 6
    assert all(r[3] and r[4] == 6 for r in res)
