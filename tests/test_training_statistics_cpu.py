"""CPU: the command line and the log of the step's optional statistics."""
import pytest


@pytest.mark.parametrize('args', [['--label-top', '65'], ['--label-top', '-1'], ['-K', '8', '--label-top', '9']], ids=' '.join)
def test_command_line_refuses_more_alternatives_than_there_are(args, capsys):
    import train
    with pytest.raises(SystemExit):
        train.parse(['--gan-type', 'StyleGAN2'] + args)
    assert '--label-top' in capsys.readouterr().err
    assert train.parse(['--gan-type', 'StyleGAN2', '-K', '8', '--label-top', '8']).label_top == 8
    assert train.parse(['--gan-type', 'StyleGAN2', '--label-top', '64']).label_top == 64


def test_the_log_shows_the_optional_statistics(tmp_path, capsys, monkeypatch):
    import types
    from warpedganspace_amd import trainer as T
    p = types.SimpleNamespace(tensorboard=False, batch_size=4, max_iter=10)
    tr = T.Trainer(params=p, exp_dir='exp', root=str(tmp_path))
    stats = {'accuracy': 0.5, 'classification_loss': 1.0, 'regression_loss': 0.25, 'total_loss': 1.25}
    moved = []
    monkeypatch.setattr(T, 'update_stdout', moved.append)
    tr.log_progress(1, 0.1, 1.0, 9.0, stats)
    plain = capsys.readouterr().out
    monkeypatch.setattr(T.sys.stdout, 'isatty', lambda: True, raising=False)
    tr.log_progress(2, 0.1, 1.0, 9.0, dict(stats, entropy=2.125, top5_accuracy=0.75))
    more = capsys.readouterr().out
    assert 'ntropy' not in plain and '2.125' in more and 'Entropy' in more and 'Top5 accuracy' in more and '0.75' in more
    assert len(more.splitlines()) == len(plain.splitlines()) + 2
    assert moved[-1:] == [12]                   # the block that the next log overwrites


def test_moments_of_another_optimizer_are_not_dropped_without_a_word(tmp_path, capsys):
    import types
    from warpedganspace_amd.trainer import Trainer
    tr = Trainer(params=types.SimpleNamespace(tensorboard=False), exp_dir='exp', root=str(tmp_path))
    engine = types.SimpleNamespace(optimizer='muon', bucket=types.SimpleNamespace(step_count=7), load_optim_state=lambda st: st.get('optimizer') == 'muon')
    tr.restore_optim(engine)
    assert capsys.readouterr().out == ''
    tr.resume_optim = {'optimizer': 'muon'}
    tr.restore_optim(engine)
    assert 'Restored momentum and Adam moments (step 7)' in capsys.readouterr().out
    tr.resume_optim = {'step': 3}               # written before the key existed: Adam's
    tr.restore_optim(engine)
    out = capsys.readouterr().out
    assert 'optimizer adam' in out and 'optimizer muon' in out and 'fresh' in out


def test_gloo_is_given_host_tensors_only(monkeypatch):
    """A stand-in for a device tensor: the collective gets its copy in host memory, and the result is copied back."""
    import torch
    from warpedganspace_amd import trainer as T
    calls = []

    class OnDevice:
        is_cuda = True

        def __init__(self, v):
            self.v = v

        def detach(self):
            return self

        def cpu(self):
            return self.v.clone()

        def copy_(self, h):
            self.v = h.clone()

    def reduce(t, op=None, async_op=False):
        calls.append((type(t), async_op))
        if isinstance(t, torch.Tensor):
            t *= 3
        return 'work' if async_op else None

    def spread(t, src):
        calls.append((type(t), src))
        if isinstance(t, torch.Tensor):
            t.fill_(7)
    backend = ['gloo']
    monkeypatch.setattr(T.dist, 'get_backend', lambda: backend[0])
    monkeypatch.setattr(T.dist, 'all_reduce', reduce)
    monkeypatch.setattr(T.dist, 'broadcast', spread)
    d = OnDevice(torch.tensor([1.0, 2.0]))
    T.all_reduce(d)
    assert d.v.tolist() == [3.0, 6.0]
    T.all_reduce(d, async_op=True).wait()
    assert d.v.tolist() == [9.0, 18.0]
    T.broadcast(d, 0)
    assert d.v.tolist() == [7.0, 7.0] and calls == [(torch.Tensor, False), (torch.Tensor, False), (torch.Tensor, 0)]
    del calls[:]
    h = torch.ones(2)
    assert T.all_reduce(h, async_op=True) == 'work'                  # host tensors and RCCL: as they are
    backend[0] = 'nccl'
    T.all_reduce(d)
    T.broadcast(d, 1)
    assert calls == [(torch.Tensor, True), (OnDevice, False), (OnDevice, 1)]
