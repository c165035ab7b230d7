"""What the C entries of the 8-bit expert products refuse on the host, at the ends of their sizes (16: non-null stand-ins that are never dereferenced)."""
from moe_distributed_training_amd._lib import lib


def test_rows_of_no_columns_need_their_scales_only():
    q = lib.moe_quantize_rows
    assert q(None, 0, 0, None, 0, None, 0, 0, None) == 0                      # no rows
    assert q(None, 0, 0, None, 0, None, 4, 0, None) == -1                     # rows, but nowhere for their scales
    assert q(None, 0, 0, None, 16, 16, 4, 0, None) == -1                      # columns of padding, but nowhere for them
    assert q(None, 8, 0, 16, 16, 16, 4, 8, None) == -1 and q(16, 8, 0, None, 16, 16, 4, 8, None) == -1
