"""CPU: limits of the training operators' C entry points that the host checks before a launch."""
import struct

import pytest

from tests.test_operator_refusals_cpu import matrix, ortho, refused

NONE = 4096        # an address that is never dereferenced: the call is refused first


def with_joined(n, **k):
    m = matrix(**k)
    return m[:-4] + struct.pack('=i', n)


@pytest.mark.parametrize('step', [False, True])
def test_joined_iterations(step):
    refused(ortho(with_joined(-1), step=step), b'joined')
    refused(ortho(with_joined(17), step=step), b'joined')
    refused(ortho(with_joined(2), with_joined(3), step=step), b'joined')
