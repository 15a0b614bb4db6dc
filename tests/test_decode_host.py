"""What the decode operators' binding and the decoder refuse or work out on the host: no GPU."""
import pytest

import b2q
from b2q.decode import Decoder

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("rows", [-1, 0, 9, 1000])
def test_a_step_refuses_rows_that_its_buffers_do_not_hold(rows):
    dec = Decoder.__new__(Decoder)   # before anything is looked up or launched
    dec.max_rows = 8
    with pytest.raises(b2q.B2QError) as e:
        dec.step(rows)
    assert e.value.status == b2q.ERR_SHAPE
