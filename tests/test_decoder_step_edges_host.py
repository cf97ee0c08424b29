"""More of the host side of sampling, without a GPU: the widest rows."""
import pytest

from shorokoo_b200 import _native
from test_decoder_step_host import _sample

L = _native.lib()


@pytest.mark.parametrize("elem", [1, 10, 16])
def test_the_widest_rows_of_logits(elem):
    """A kernel's sums hold the weights of 2^21 logits; one more is refused."""
    assert _sample(elem=elem, rows=0, vocab=1 << 21) == 0
    for rows in (0, 1):
        assert _sample(elem=elem, rows=rows, vocab=(1 << 21) + 1) == 2
        assert "2097153" in L.sb_last_error().decode()
