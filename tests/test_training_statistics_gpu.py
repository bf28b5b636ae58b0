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
