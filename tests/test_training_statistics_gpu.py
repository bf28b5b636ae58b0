"""The step's optional statistics: what is refused, and what reading them costs."""
import pytest

from tests.test_muon_training_gpu import batch, make

pytestmark = pytest.mark.gpu


def test_more_alternatives_than_there_are_paths_are_refused(dev):
    for bad in (17, 65, -1):
        with pytest.raises(ValueError, match='label_top'):
            make(dev, label_top=bad)
    eng = make(dev, label_top=16)
    eng.step(*batch(dev, 1))
    assert eng.pop_stats()['top16_accuracy'] == 1.0


def test_statistics_are_read_in_one_transfer(dev, monkeypatch):
    import torch
    eng = make(dev, lambda_ent=0.1, label_top=3)
    eng.step(*batch(dev, 1))
    want = torch.cat([eng.stats_sum, eng.extra_sum]).tolist()
    reads = []
    tolist = torch.Tensor.tolist
    monkeypatch.setattr(torch.Tensor, 'tolist', lambda t: reads.append(t.shape) or tolist(t))
    got = eng.pop_stats()
    assert len(reads) == 1
    assert [got[k] for k in ('classification_loss', 'regression_loss', 'total_loss', 'accuracy', 'entropy', 'top3_accuracy')] == want
    assert eng.pop_stats() == dict.fromkeys(got, 0.0)
