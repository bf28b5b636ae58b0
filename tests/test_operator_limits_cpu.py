"""CPU: what the host checks of the training operators' arguments before a launch, beyond the plain refusals."""
import random
import struct

import pytest

from tests.test_operator_refusals_cpu import I64, P, matrix, ortho, refused
from warpedganspace_amd import _lib as L
from warpedganspace_amd import ops


def with_joined(n, **k):
    m = matrix(**k)
    return m[:-4] + struct.pack('=i', n)


@pytest.mark.parametrize('step', [False, True])
def test_joined_iterations(step):
    refused(ortho(with_joined(-1), step=step), b'joined')
    refused(ortho(with_joined(17), step=step), b'joined')
    refused(ortho(with_joined(2), with_joined(3), step=step), b'joined')


def _span(base, rows, cols, offset, stride, written=True, size=4):
    return (base + offset * size, 1, rows * cols * size, rows * cols * size, written) if stride == cols else (base + offset * size, rows, cols * size, stride * size, written)


def _elements(rows, cols, offset, stride):
    return {offset + r * stride + c for r in range(rows) for c in range(cols)}


def _refused(*views, written=(True, True, True)):
    try:
        ops._check_apart([_span(4096, *v, written=w) for v, w in zip(views, written)])
    except L.WgsError as e:
        assert 'overlaps' in str(e)
        return True
    return False


def test_overlaps_of_strided_weights_are_refused():
    """Views (rows, columns, offset, row stride) of one storage."""
    assert _refused((8, 5, 0, 10), (4, 5, 60, 10))          # rows 0 .. 7 and 6 .. 9 of the same columns
    assert _refused((4, 10, 0, 20), (4, 10, 5, 20))         # columns 0 .. 9 and 5 .. 14
    assert _refused((8, 5, 0, 10), (1, 5, 30, 5))           # a single row inside
    assert _refused((8, 5, 0, 10), (2, 10, 38, 10))         # a dense part across a row's end
    assert _refused((8, 5, 0, 10), (3, 5, 16, 15))          # other strides
    assert not _refused((8, 5, 0, 10), (8, 5, 5, 10))       # the other columns
    assert not _refused((4, 5, 0, 10), (4, 5, 40, 10))
    assert not _refused((8, 5, 0, 10), (1, 5, 35, 5))       # between two rows
    assert not _refused((8, 5, 0, 10), (4, 5, 5, 20))       # every other gap
    assert not _refused((8, 5, 0, 10), (8, 5, 0, 10), written=(False, False))      # gradients may be shared
    assert _refused((8, 5, 0, 10), (8, 5, 0, 10), written=(True, False))
    assert _refused((8, 5, 0, 10), (8, 5, 0, 10), written=(False, True))
    assert _refused((2, 50, 0, 200), (1, 10, 10, 10), written=(False, True)) and not _refused((2, 50, 0, 200), (1, 10, 60, 10), written=(False, True))


def test_overlaps_against_the_sets_of_elements():
    rng = random.Random(0)
    met = 0
    for _ in range(4000):
        views = []
        for _ in range(2):
            cols = rng.randint(1, 6)
            views.append((rng.randint(1, 6), cols, rng.randint(0, 40), rng.choice([cols, cols + 1, 7, 8, 12, 13])))
        want = bool(_elements(*views[0]) & _elements(*views[1]))
        assert _refused(*views) == want, views
        met += want
    assert 500 < met < 3500


def test_three_spans_of_which_the_outer_ones_overlap():
    """The middle one lies in a gap and ends before the last one starts."""
    assert _refused((4, 5, 0, 20), (1, 5, 6, 5), (1, 5, 44, 5))
    assert not _refused((4, 5, 0, 20), (1, 5, 6, 5), (1, 5, 45, 5))


@pytest.mark.parametrize('order', [1, -1])
def test_a_large_matrix_beside_a_long_batch_of_small_ones_is_cut_into_runs(order):
    """All matrices of a run have as many partial norms (16 bytes each) as its largest: 256 for 2048 x 2048, in at most 2^22 workgroups."""
    lib = L.lib()
    big, small = matrix(2048, 2048, rs=2048, bs=1 << 22, obs=1 << 22), matrix(17, 17, 70000, rs=17, bs=289, obs=289)

    def need(*m):
        return lib.wgs_orthogonalise_ws_bytes(b''.join(m[::order]), len(m), 0, 5)
    one = need(matrix(17, 17, 1, rs=17, bs=289, obs=289))
    assert need(small) < 70000 * (one + 64)                          # one partial norm each: a single run
    # in the large one's run at most 2^14 instances; the rest goes without it
    assert need(big, small) <= max(need(big) + (1 << 14) * (one + 64) + (16 << 22), need(small))


def test_label_logprobs_backward_refuses_more_workgroups_than_a_grid_holds():
    """256 threads a workgroup, fewer than 2^32 threads a grid: 2^23 rows of two parts (over 1024 16-byte vectors) are too many."""
    def bwd(rows, V):
        return L.lib().wgs_label_logprobs_bwd(P, 1, I64(rows), I64(V), I64(V), P, I64(-100), P, P, 0, None, P, None, None, P, I64(V), None)
    refused(bwd(1 << 23, 8200), b'too many scores')
    refused(bwd((1 << 24) - 1, 16384), b'too many scores')
