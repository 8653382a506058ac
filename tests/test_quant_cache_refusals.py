"""What the quantised cache refuses before anything is launched (no GPU needed), and what it says then."""
import pytest

from test_attention_refusals import FAKE, attend, geom, qgeom


@pytest.mark.parametrize("n", [2 ** 33, 2 ** 40, 2 ** 62, 2 ** 63 - 1])
def test_more_rows_than_one_call_takes(n):
    """Refused with a text of its own, not with that of an earlier call; no count wraps."""
    from ucmx import _native as N
    assert attend(q=0) == N.EPARAM
    before = N.last_error()
    assert N.lib.ucmx_quant_write_tokens(FAKE, FAKE, 256, 256, n, FAKE, FAKE, qgeom(), None) == N.EUNSUPPORTED
    assert "rows" in N.last_error() and N.last_error() != before


def test_more_blocks_than_one_call_takes():
    from ucmx import _native as N
    T, H = 1 << 20, 1 << 16
    kg = geom(block_tokens=T, n_kv_heads=H, token_stride=H * 128, block_stride=T * H * 128)
    g = qgeom(block_tokens=T, n_kv_heads=H, block_stride=H * (T // 16) * 2176)
    assert attend(q=0) == N.EPARAM
    assert N.lib.ucmx_quant_write_blocks(FAKE, kg, FAKE, kg, FAKE, None, 2 ** 31 - 1, FAKE, g, None) == N.EUNSUPPORTED
    assert "rows" in N.last_error()
    assert attend(q=0) == N.EPARAM
    assert N.lib.ucmx_quant_read_blocks(FAKE, g, FAKE, None, 2 ** 31 - 1, FAKE, kg, FAKE, kg, None) == N.EUNSUPPORTED
    assert "rows" in N.last_error()
