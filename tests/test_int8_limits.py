"""What the C entries of the 8-bit expert products refuse on the host, at the ends of their sizes (16: non-null stand-ins that are never dereferenced)."""
from moe_distributed_training_amd._lib import lib


def test_rows_of_no_columns_need_their_scales_only():
    q = lib.moe_quantize_rows
    assert q(None, 0, 0, None, 0, None, 0, 0, None) == 0                      # no rows
    assert q(None, 0, 0, None, 0, None, 4, 0, None) == -1                     # rows, but nowhere for their scales
    assert q(None, 0, 0, None, 16, 16, 4, 0, None) == -1                      # columns of padding, but nowhere for them
    assert q(None, 8, 0, 16, 16, 16, 4, 8, None) == -1 and q(16, 8, 0, None, 16, 16, 4, 8, None) == -1


def test_more_threads_than_a_grid_counts_are_refused():
    """A launch's threads are counted in 32 bits: rows beyond that are refused before anything is enqueued, whatever the launch that has too many."""
    unsupported, rows = -2, 1 << 24                                            # 2^24 rows of 256 threads
    assert lib.moe_quantize_rows(16, 4096, 0, 16, 4096, 16, rows, 4096, None) == unsupported
    assert lib.moe_quantize_rows(16, 20000, 0, 16, 20096, 16, 1 << 22, 20000, None) == unsupported       # 1024 threads
    assert lib.moe_combine_f32(16, 8, 16, 8, 0, None, 0, 2, rows, 8, None) == unsupported
    assert lib.moe_combine_f32_dgates(16, 8, 16, 8, 0, 16, 0, 4, rows // 4, 8, None) == unsupported
    n = 1 << 50
    big = 1 << 26
    assert lib.moe_linear_int8_fwd(16, 64, big, 0, 16, 8192, 1, 64, 16, 16, 128, 0, 16, 0, 16, 0, 2, big, 64, 128, 1, 1, 1, 16, n, None) == unsupported
    assert lib.moe_linear_int8_bwd(16, 128, 0, 1, 1, None, 0, 16, 8192, 1, 64, 16, 16, 64, 0, 1, 16, 0, 16, 0, 2, big, 64, 128, 16, n, None) == unsupported
    # few rows to code, but tiles of so many columns
    assert lib.moe_linear_int8_fwd(16, 64, 1 << 21, 0, 16, 1 << 30, 1, 64, 16, 16, 1 << 24, 0, 16, 0, 16, 0, 1, 1 << 21, 64, 1 << 24, 1, 1, 1, 16, n, None) == unsupported
    # strided weights of more columns than the copy's grid has
    assert lib.moe_linear_int8_fwd(16, 16, 8, 0, 16, 1, 3, 48, 16, 16, 1 << 23, 0, 16, 0, 16, 0, 1, 8, 16, 1 << 23, 1, 1, 1, 16, n, None) == unsupported

    def mlp(R, f, x_rows):
        return lib.moe_mlp_int8_fwd(16, 64, x_rows, 0, 16, 16, 16, 16, 16, 16, 16, 64, 0, 16, 0, 16, 0, 2, R, 64, f, R // x_rows, 0, None, 0, 16, n, None)
    assert mlp(rows, 2048, rows // 64) == unsupported                          # codes of h

    def mlp_bwd(R, f):
        return lib.moe_mlp_int8_bwd(16, 64, 0, 0, 1, None, 0, 16, 16, 16, 16, 16, 16, 16, n, 16, 64, 0, 16, 0, 16, 0, 2, R, 64, f, 16, n, None)
    assert mlp_bwd(1 << 23, 8192) == unsupported                               # codes of dgate and dup, 512 threads
