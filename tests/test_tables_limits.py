"""Sizes that the tables' kernels do not count in 32 bits are refused; no device needed."""
import pytest

from kyro_amd import _lib
from tests.test_request_tables import CALLS, call

MOST = 2 ** 31 - 2048


@pytest.mark.parametrize("name", sorted(CALLS))
def test_sizes_past_the_kernels_arithmetic(name):
    far = dict({k: i << 50 for i, k in enumerate(CALLS[name], 1)}, block_size=1, num_blocks=2 ** 31 - 1)  # arrays far apart
    for change, text in ((dict(max_state_blocks=MOST + 1, **far), "blocks"), (dict(batch_size=2 ** 24, **far), "one launch"),
                         (dict(batch_size=2 ** 31 - 1, **far), "one launch")):
        rc, msg = call(name, **change)
        assert rc == _lib.KYRO_EUNSUPPORTED and text in msg and "tables_" + name in msg, msg
    rc, msg = call(name, max_state_blocks=MOST, **far)
    assert rc == _lib.KYRO_EINVAL and "null kyro_ctx" in msg, msg


def test_widths_of_extend():
    rc, msg = call("extend", max_blocks_per_seq=MOST + 1, block_table=1 << 50)
    assert rc == _lib.KYRO_EUNSUPPORTED and "blocks" in msg, msg
    rc, msg = call("extend", max_blocks_per_seq=MOST, block_table=1 << 50)
    assert rc == _lib.KYRO_EINVAL and "null kyro_ctx" in msg, msg
    rc, msg = call("keep", max_blocks_per_seq=2 ** 31 - 1)  # not read
    assert rc == _lib.KYRO_EINVAL and "null kyro_ctx" in msg, msg
