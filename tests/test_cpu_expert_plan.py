"""Which operands of an expert product are copied to rows of whole chunks first, as the workspace's size says."""

from apexw_amd import _lib

OK = 4096        # an aligned address: nothing is launched here
NK, KN = _lib.EXPERT_NK, _lib.EXPERT_KN


def rows_bytes(lda, ldw, order, rows, k, n, experts=1):
    sw = (n if order == NK else k) * ldw
    return _lib.load().apexw_expert_rows_workspace(OK, lda, OK, ldw, sw, order, experts, rows, k, n)


def weight_bytes(ld_dy, ld_x, rows, n, k, experts=1):
    return _lib.load().apexw_expert_weight_grad_workspace(OK, ld_dy, OK, ld_x, experts, rows, n, k)


def test_overlapping_k_rows_are_copied():
    """Rows of k closer than their width: both operands of a weight grad and [k][n] weights, nothing else."""
    n, k, rows = 4096, 2048, 8192
    assert weight_bytes(n, k, rows, n, k) == 0
    assert weight_bytes(0, k, rows, n, k) == 2 * rows * n
    assert weight_bytes(n, 8, rows, n, k) == 2 * rows * k
    assert weight_bytes(n - 8, k - 8, rows, n, k) == 2 * rows * (n + k)
    assert rows_bytes(k, n, KN, rows, k, n) == 0
    assert rows_bytes(k, n - 8, KN, rows, k, n) == 2 * k * n
    assert rows_bytes(0, k, NK, rows, k, n) == 0 and rows_bytes(k, 0, NK, rows, k, n) == 0


def test_copies_keep_to_32_bit_offsets():
    """Rows wider than 2^22 elements are not copied, whatever would be gained: a copy's rows are as far apart."""
    most = 1 << 22
    assert weight_bytes(8 * most, 16, 64, most, 16) == 2 * 64 * most        # far apart, not wide: copied
    assert weight_bytes(most - 1, 16, 64, most - 1, 16) == 2 * 64 * most
    for n in (most + 1, most + 8, 36_000_001, 40_000_000):
        assert weight_bytes(n, 16, 64, n, 16) == 0 and weight_bytes(16, n, 64, 16, n) == 0
    # rows products: what is left is a general product in parts, or whole
    wide, parts = most + 1, 64 * 4096 * 16 * 4
    assert rows_bytes(most - 1, most - 1, NK, 4096, most - 1, 16) >= 2 * 4096 * most
    assert rows_bytes(wide, wide, NK, 4096, wide, 16) <= parts < 2 * 4096 * most
    assert rows_bytes(16, most - 1, KN, 4096, 16, most - 1) >= 2 * 16 * most
    assert rows_bytes(16, wide, KN, 4096, 16, wide) == 0
