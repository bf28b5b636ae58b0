"""GPU, world_size 2: the data-parallel branches of TrainStep itself (lib/trainer.py:162-166 is nn.DataParallel in the
reference; here one process per rank).

Two processes share cuda:0 (RCCL refuses two ranks on one device, so the process group is gloo, which all-reduces device
tensors through host staging — the collective calls, streams and ordering in TrainStep.step are the ones the RCCL run
uses).  Each rank first runs the SAME shard through a world=1 engine, then through a world=2 engine built from identical
weights; checked:
  * replicas start from rank 0's parameters (rank 1 is built from different random weights on purpose);
  * the all-reduced gradient bucket == sum of the two ranks' world=1 gradients (DataParallel semantics: per-rank
    BatchNorm statistics, loss = mean over the global batch <=> mean of the ranks' means);
  * post-Adam parameters == Adam on the averaged gradient, identical on both ranks;
  * pop_stats() averages over ranks; the per-rank sampler draws different z on the two ranks.
"""
import os
import socket
import types

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

pytestmark = pytest.mark.gpu


def _failure_text(r):
    """what a failed launcher run said: the lines that name a cause (a rank's traceback, a GPU memory fault, an HSA status) from anywhere in
    its stderr — the runtime's queue dump behind a fault is thousands of lines long and used to push them out of the tail — then the tails"""
    import re
    key = [ln for ln in r.stderr.splitlines() if re.search(r'fault|HSA_STATUS|hipError|Traceback|Error:|error:|Aborted|out of memory', ln)]
    return '\n'.join(key[:40]) + '\n--- stdout tail ---\n' + r.stdout[-1500:] + '\n--- stderr head ---\n' + r.stderr[:1500] + '\n--- stderr tail ---\n' + r.stderr[-1500:]


def _run_launcher(cmd, timeout, repo):
    """bench.py through its launcher with N rank processes."""
    import subprocess
    return subprocess.run(cmd, capture_output=True, text=True, timeout=timeout, env=dict(os.environ, PYTHONPATH=repo))


# Rank processes that share ONE GPU under the launcher: about one run in twenty lost a rank to HSA_STATUS_ERROR_ILLEGAL_INSTRUCTION while gloo
# all-reduced device tensors (1 / 20 and 1 / 12 with eight ranks, 3 / 6 on one box; never with one process per GPU, never without collectives).  The
# collectives go through host memory since (trainer.all_reduce), but that they were the cause is not shown: the case stays off.
_shared_gpu_abort = pytest.mark.skip(reason='rank processes sharing one GPU under the launcher have lost a rank to HSA_STATUS_ERROR_ILLEGAL_INSTRUCTION; '
                                            'the cause is not shown')


def _free_port():
    s = socket.socket()
    s.bind(('127.0.0.1', 0))
    p = s.getsockname()[1]
    s.close()
    return p


def _build(dev, seed_r, world, rank, B, K=16, N=4, size=32):
    from tests import golden_inputs as GI
    from warpedganspace_amd.gan_load import StyleGAN2Wrapper
    from warpedganspace_amd.reconstructor import Reconstructor
    from warpedganspace_amd.stylegan2 import Generator
    from warpedganspace_amd.support_sets import SupportSets
    from warpedganspace_amd.trainer import TrainStep
    torch.manual_seed(0)
    G = Generator(size, 512, 8)
    sd_g = GI.fill_state_dict(G.state_dict(), 900 + size)
    for k in sd_g:
        if k.startswith('style.') and k.endswith('weight'):
            sd_g[k] = sd_g[k] * 100.0
    G.load_state_dict(sd_g)
    c = GI.support_sets_case(K, N, 512, 2 * B, 31, learn_gammas=True)
    S = SupportSets(K, N, 512, learn_gammas=True, gamma=c['gamma'])
    S.load_state_dict(c['sd'])
    torch.manual_seed(seed_r)                  # R's constructor initialisation
    R = Reconstructor('ResNet', K)
    params = types.SimpleNamespace(reconstructor_lr=1e-4, support_set_lr=1e-4, min_shift_magnitude=0.25,
                                   max_shift_magnitude=0.45, lambda_cls=1.0, lambda_reg=0.25, z_truncation=None,
                                   shift_in_w_space=False)
    eng = TrainStep(StyleGAN2Wrapper(G, False).to(dev).eval(), S.to(dev).train(), R.to(dev).train(), params, B, dev,
                    world=world, seed=5, rank=rank)
    return eng, c


def _worker(rank, world, port, q):
    try:
        os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port), HSA_ENABLE_IPC_MODE_LEGACY='0')
        torch.cuda.set_device(0)
        dev = torch.device('cuda', 0)
        dist.init_process_group('gloo', rank=rank, world_size=world)
        B = 2
        # --- world=1 engines on this rank's shard, from rank 0's weights (seed 11 on both ranks)
        e1, c = _build(dev, 11, 1, 0, B)
        sl = slice(rank * B, (rank + 1) * B)
        z, idx = c['z'][sl].to(dev), c['idx'][sl].to(dev)
        mag = torch.tensor([0.3, -0.4, 0.35, 0.28])[sl].to(dev)
        p0 = e1.bucket.flat.clone()

        def warm(e):     # build the generator's lazy weight caches, then take the two-stream schedule of a steady-state step
            with torch.no_grad():    # (un-shifted pass, deferred weight gradients and R's all-reduce on the side stream)
                e.G(z)
            torch.cuda.synchronize()
            e.steps_done = 1
        warm(e1)
        st1 = e1.step(z, idx, mag).clone()
        g_local = e1.bucket.grad.clone()
        # --- world=2 engine; rank 1 deliberately starts from DIFFERENT reconstructor weights
        e2, _ = _build(dev, 11 + rank, world, rank, B)
        assert torch.equal(e2.bucket.flat, p0), "replicas must start from rank 0's parameters"
        e2.comm_events = []
        warm(e2)
        e2.step(z, idx, mag)
        torch.cuda.synchronize()
        g_sum = e2.bucket.grad.clone()
        expect = g_local.clone()
        dist.all_reduce(expect)
        scale = float(expect.abs().max())
        err_g = float((g_sum - expect).abs().max()) / scale
        # Adam on the averaged gradient (first step: m = (1-b1) g, v = (1-b2) g^2, bias-corrected)
        g = (expect / world).double()
        upd = torch.zeros_like(g)
        for lr, a, b in e2.bucket.groups:
            gg = g[a:b]
            upd[a:b] = lr * gg / (gg.abs() + 1e-8)
        p_expect = p0.double() - upd
        big = g.abs() > 1e-3 * g.abs().max()           # entries with a numerically meaningful gradient
        err_p = float((e2.bucket.flat.double() - p_expect)[big].abs().max())
        # both ranks hold the same parameters after the step
        mine = e2.bucket.flat.clone()
        other = mine.clone()
        dist.broadcast(other, 0)
        same = bool(torch.equal(mine, other))
        # statistics are averaged over ranks
        st = e2.pop_stats()
        tot = st1[2:3].clone()
        dist.all_reduce(tot)
        err_s = abs(st['total_loss'] - float(tot) / world)
        # per-rank sampler: different z on the two ranks, same on a re-built engine with the same (seed, rank)
        zs, _, _ = e2.sample()
        zo = zs.clone()
        dist.broadcast(zo, 0)
        differs = (rank == 0) or (not torch.equal(zs, zo))
        n_ev = len(e2.comm_events)
        q.put((rank, err_g, err_p, same, err_s, differs, n_ev, e2.allreduce_bytes, None))
        dist.barrier()
        dist.destroy_process_group()
    except Exception as e:  # noqa: BLE001
        import traceback
        q.put((rank, None, None, None, None, None, None, None, traceback.format_exc()))
        raise


@pytest.mark.timeout(900)
def test_trainstep_world2_matches_sum_of_rank_gradients(dev):
    world = 2
    ctx = mp.get_context('spawn')
    torch.cuda.empty_cache()                 # the two ranks share this device with the test process's cached blocks

    def run():
        port = _free_port()
        q = ctx.SimpleQueue()
        procs = [ctx.Process(target=_worker, args=(r, world, port, q)) for r in range(world)]
        for p in procs:
            p.start()
        res = [q.get() for _ in range(world)]
        for p in procs:
            p.join(120)
        return res, procs
    res, procs = run()
    # one retry for rendezvous trouble only (a port taken between _free_port() and the bind, a gloo connect timeout):
    # a failed comparison is reported by the asserts below, never retried
    if any(r[-1] is not None and any(s in r[-1] for s in ('Address already in use', 'timed out', 'Connection', 'connect')) for r in res):
        print('rendezvous failed, retrying once:', [r[-1].splitlines()[-1] for r in res if r[-1]])
        res, procs = run()
    for r in res:
        assert r[-1] is None, r[-1]
    for rank, err_g, err_p, same, err_s, differs, n_ev, nbytes, _ in res:
        print('rank %d: grad err %.2e, param err %.2e, stats err %.2e, all-reduce payload %d B' % (rank, err_g, err_p, err_s, nbytes))
        assert err_g < 2e-5, err_g           # wgrad split-K atomics reorder fp32 sums between the two runs
        assert err_p < 2e-6, err_p           # |update| = lr = 1e-4 per entry
        assert same
        assert err_s < 1e-5
        assert differs
        assert n_ev == 1 and nbytes > 0
    assert all(p.exitcode == 0 for p in procs)


def _bench_two_ranks(backend, tmp_path):
    import json
    import subprocess
    import sys
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    side = str(tmp_path / 'bench_extra.json')
    cmd = [sys.executable, os.path.join(repo, 'bench.py'), '--gpus', '2', '--dist-backend', backend, '--steps', '3', '--warmup', '2', '--batch', '4',
           '--size', '32', '-K', '16', '-N', '4', '--no-cpu-baseline', '--no-extra', '--extra-out', side]
    r = _run_launcher(cmd, 600, repo)
    assert r.returncode == 0, _failure_text(r)
    lines = [ln for ln in r.stdout.splitlines() if ln.startswith('{')]
    assert len(lines) == 1, r.stdout[-2000:]                  # rank 0 alone prints the record
    assert len(lines[0]) < 4096                               # the driver keeps ~8 KB of stdout: the N > 1 line obeys the size cap too
    d = json.loads(lines[0])
    assert d['n_gpus'] == 2 and d['steps'] == 3 and d['warmup'] == 2 and d['scaling'] == 'weak' and d['dtype'] == 'fp32'
    assert d['config']['global_batch'] == 8 and d['config']['parallelism'] == 'dp2'
    assert abs(d['value'] - 8 * 3 / (d['ms_per_step'] * 3e-3)) < 0.02 * d['value']          # whole-job rate over both ranks
    c = d['comm']
    assert c['world_size_observed'] == 2 and c['collectives_per_step'] == 2 and c['allreduce_bytes_per_step'] > 0 and c['exposed_wait_ms_per_step'] >= 0
    assert d['roofline']['kernel'] and 0 <= d['roofline']['frac'] <= 1.0 and d['host']['library_launches_per_step'] > 0
    assert d['product']['value'] > 0 and d['direct_fp32']['precision'] == 'fp32' and d['config']['precision'] == 'fp32w'
    full = json.load(open(side))                               # the side file holds the complete records
    e = full['extra'][0]
    assert e['n_gpus'] == 2 and e['steps'] == 3 and e['comm']['world_size_observed'] == 2 and e['roofline']['kernel']
    assert full['extra'][1]['precision'] == 'fp32' and full['extra'][1]['n_gpus'] == 2     # the direct-form run beside it
    return d


@_shared_gpu_abort
def test_bench_two_ranks_end_to_end_over_gloo(tmp_path):
    """`bench.py --gpus 2 --dist-backend gloo`: the driver's N > 1 invocation end to end on ONE device (rank spawn, process
    group, per-rank engines, barrier + max-over-ranks timing, comm section, the product / direct runs at N = 2, rank-0 JSON) — so that
    the first RCCL run of the scaling bench is not also this code path's first run."""
    d = _bench_two_ranks('gloo', tmp_path)
    assert d['comm']['backend'].startswith('gloo')


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason='RCCL needs one GPU per rank: runs where >= 2 GPUs are visible')
def test_bench_two_ranks_end_to_end_over_rccl(tmp_path):
    """The same on RCCL (`nccl` backend, one rank per GPU) wherever the box has two GPUs: the driver's multi-GPU scaling run is then
    never RCCL's first contact with this code."""
    d = _bench_two_ranks('nccl', tmp_path)
    assert d['comm']['backend'].startswith('RCCL')


class _FakeWriter:
    def __init__(self):
        self.rows = []

    def add_scalar(self, key, value, it):
        self.rows.append((key, it))


def _train_worker(rank, world, port, root, q):
    try:
        from warpedganspace_amd.gan_load import build_stylegan2
        from warpedganspace_amd.reconstructor import Reconstructor
        from warpedganspace_amd.support_sets import SupportSets
        from warpedganspace_amd.trainer import Trainer
        os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port), HSA_ENABLE_IPC_MODE_LEGACY='0')
        torch.cuda.set_device(0)
        dist.init_process_group('gloo', rank=rank, world_size=world)
        log_freq = 3
        p = types.SimpleNamespace(reconstructor_lr=1e-4, support_set_lr=1e-4, min_shift_magnitude=0.25, max_shift_magnitude=0.45,
                                  lambda_cls=1.0, lambda_reg=0.25, z_truncation=None, shift_in_w_space=False, tensorboard=False,
                                  log_freq=log_freq, ckp_freq=1000, max_iter=2 * log_freq, batch_size=4, seed=3, precision='fp32')
        torch.manual_seed(0)
        G = build_stylegan2(None, resolution=32)
        S = SupportSets(8, 4, 512, learn_alphas=False, learn_gammas=True, gamma=1.0 / 512)
        R = Reconstructor('ResNet', 8)
        tr = Trainer(params=p, exp_dir='exp', use_cuda=True, root=os.path.join(root, 'r%d' % rank))
        n_pop = [0]
        if rank == 0:
            tr.tb_writer = _FakeWriter()         # `--tensorboard` as it lands: rank 0 owns the only writer
        eng = tr.train(G, S, R)
        flat = eng.bucket.flat.clone()
        other = flat.clone()
        dist.broadcast(other, 0)
        q.put((rank, tr.tb_active, len(tr.tb_writer.rows) if rank == 0 else 0, bool(torch.equal(flat, other)), eng.steps_done, None))
        dist.barrier()
        dist.destroy_process_group()
    except Exception:  # noqa: BLE001
        import traceback
        q.put((rank, None, None, None, None, traceback.format_exc()))
        raise


@pytest.mark.timeout(900)
def test_trainer_loop_with_a_rank0_only_tensorboard_writer(dev, tmp_path):
    """Trainer.train over two ranks for 2 x log_freq iterations with a TensorBoard writer on rank 0 only (lib/trainer.py:127-131 builds it
    in every process of the reference; here rank 0's alone): pop_stats() all-reduces, so both ranks must pop in EVERY iteration — the
    loop used to test `self.tb_writer`, which differs between the ranks (mismatched collectives)."""
    world = 2
    ctx = mp.get_context('spawn')
    torch.cuda.empty_cache()
    port = _free_port()
    q = ctx.SimpleQueue()
    procs = [ctx.Process(target=_train_worker, args=(r, world, port, str(tmp_path), q)) for r in range(world)]
    for p in procs:
        p.start()
    for p in procs:
        p.join(600)
    alive = [p for p in procs if p.is_alive()]
    for p in alive:
        p.kill()
    assert not alive, "ranks hung: mismatched collectives"
    res = sorted(q.get() for _ in range(world))
    for r in res:
        assert r[-1] is None, r[-1]
    assert [r[1] for r in res] == [True, True]
    assert res[0][2] == 4 * 6                      # four scalars in each of the 2 x log_freq iterations
    assert all(r[3] for r in res) and all(r[4] == 6 for r in res)      # replicas identical after the run
    assert all(p.exitcode == 0 for p in procs)


@_shared_gpu_abort
def test_bench_eight_ranks_end_to_end_over_gloo(tmp_path):
    """`bench.py --gpus 8 --dist-backend gloo` on ONE device with a small batch: the launcher path, eight per-rank engines, barrier +
    max-over-ranks timing and the N = 8 line (< 4 KB, comm.world_size_observed == 8, the N = 1 reference value beside the exposed wait)."""
    import json
    import subprocess
    import sys
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    side = str(tmp_path / 'bench_extra.json')
    cmd = [sys.executable, os.path.join(repo, 'bench.py'), '--gpus', '8', '--dist-backend', 'gloo', '--steps', '2', '--warmup', '1', '--batch', '2',
           '--size', '32', '-K', '16', '-N', '4', '--no-cpu-baseline', '--no-extra', '--no-direct-run', '--extra-out', side]
    r = _run_launcher(cmd, 1200, repo)
    assert r.returncode == 0, _failure_text(r)
    lines = [ln for ln in r.stdout.splitlines() if ln.startswith('{')]
    assert len(lines) == 1 and len(lines[0]) < 4096
    d = json.loads(lines[0])
    assert d['n_gpus'] == 8 and d['config']['global_batch'] == 16 and d['config']['parallelism'] == 'dp8'
    c = d['comm']
    assert c['world_size_observed'] == 8 and c['collectives_per_step'] == 2 and c['exposed_wait_ms_per_step'] >= 0
    assert c['per_gpu_images_per_sec'] > 0 and abs(c['per_gpu_images_per_sec'] * 8 - d['value']) < 0.01 * d['value'] + 0.1
    assert d['product']['value'] > 0
    full = json.load(open(side))
    assert full['host_pinning_plan'] and len(full['host_pinning_plan']) == 8          # the plan every rank would take under RCCL


def _rccl_worker(port, q):
    try:
        os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port), HSA_ENABLE_IPC_MODE_LEGACY='0')
        torch.cuda.set_device(0)
        dev = torch.device('cuda', 0)
        dist.init_process_group('nccl', rank=0, world_size=1)        # "nccl" is RCCL on ROCm
        B = 2
        e1, c = _build(dev, 11, 1, 0, B)
        z, idx = c['z'][:B].to(dev), c['idx'][:B].to(dev)
        mag = torch.tensor([0.3, -0.4]).to(dev)

        def warm(e):
            with torch.no_grad():
                e.G(z)
            torch.cuda.synchronize()
            e.steps_done = 1
        warm(e1)
        e1.step(z, idx, mag)
        torch.cuda.synchronize()
        g1 = e1.bucket.grad.clone()
        # the data-parallel branches (world = 2 as far as the engine knows) over a ONE-rank RCCL group: broadcasts, the two asynchronous
        # all-reduces (side stream / main stream), their stream-ordered wait() in front of Adam — RCCL's semantics, not gloo's host-blocking ones
        e2, _ = _build(dev, 11, 2, 0, B)
        e2.comm_events = []
        warm(e2)
        for _ in range(3):
            e2.step(z, idx, mag)
        torch.cuda.synchronize()
        e3, _ = _build(dev, 11, 2, 0, B)
        warm(e3)
        e3.step(z, idx, mag)
        torch.cuda.synchronize()
        scale = float(g1.abs().max())
        err = float((e3.bucket.grad - g1).abs().max()) / scale      # a sum over one rank: the local gradient
        st = e2.pop_stats()                                          # (an all-reduce of the statistics)
        ok = bool(torch.isfinite(e2.bucket.flat).all()) and bool(torch.isfinite(torch.tensor(list(st.values()))).all())
        waits = [a.elapsed_time(b) for a, b in e2.comm_events]
        q.put((err, ok, len(waits), e2.allreduce_bytes, dist.get_backend(), None))
        dist.barrier()
        dist.destroy_process_group()
    except Exception:  # noqa: BLE001
        import traceback
        q.put((None, None, None, None, None, traceback.format_exc()))
        raise


@pytest.mark.timeout(600)
def test_trainstep_data_parallel_branches_over_a_one_rank_rccl_group(dev):
    """RCCL contact on the one GPU this box has: the engine's world > 1 branches (parameter broadcast, the asynchronous all-reduces of R's and
    S's gradient groups, the stream-ordered wait in front of Adam, the statistics all-reduce) driven through a real `nccl` process group of
    size 1.  The sum over one rank is the local gradient: compared with the world = 1 engine's; three consecutive steps stay finite."""
    ctx = mp.get_context('spawn')
    q = ctx.Queue()
    p = ctx.Process(target=_rccl_worker, args=(_free_port(), q))
    p.start()
    err, ok, n_ev, nbytes, backend, tb = q.get(timeout=500)
    p.join(60)
    assert tb is None, tb
    print('one-rank RCCL group: gradient error vs the world-1 engine %.2e, all-reduce payload %d B per step' % (err, nbytes))
    assert backend == 'nccl' and err < 2e-5 and ok and n_ev == 3 and nbytes > 0
    assert p.exitcode == 0
