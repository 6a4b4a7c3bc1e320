"""The longest sequence that the attention over 8-bit codes takes, and how its operators trace."""
import pytest

from fa_mi355x import capi
from tests.test_quant_host import FWD


@pytest.mark.parametrize("pages,fits", [(1 << 24, True), ((1 << 24) + 1, False), ((1 << 25) - 1, False)])
def test_tokens_of_a_table_row(pages, fits):
    p = capi.new_quant_fwd_params(**dict(FWD, max_pages=pages, page_table_row_stride=pages))
    status, _ = capi.quant_fwd_workspace_size(p)
    assert status == (capi.FA_OK if fits else capi.FA_EINVAL)
    if not fits:
        assert "2^30 tokens" in capi.last_error()


def test_tokens_of_a_contiguous_sequence():
    p = capi.new_quant_fwd_params(**dict(FWD, page_table=None, num_pages=2, page_size=(1 << 30) + 64, scale_block=64))
    assert capi.quant_fwd_workspace_size(p)[0] == capi.FA_EINVAL and "2^30 tokens" in capi.last_error()
