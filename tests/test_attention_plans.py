"""CPU: the workspace that paged attention asks for (a query of sizes, no GPU call)."""
import pytest

import qlinear

MB = 1 << 20


@pytest.mark.parametrize("D", [96, 256])
@pytest.mark.parametrize("T,n", [(4096, 4096), (16384, 16384), (32768, 32768), (512, 131072), (4096, 131072), (2048, 1 << 20)])
def test_chunks_on_the_small_row_kernel_need_no_gigabytes(D, T, n):
    """Their row blocks fill the GPU; partial results of each token for each piece of 2048 positions
    were up to 13.7 GB."""
    for B in (1, 3):
        need = qlinear.paged_attention_workspace_size(B * T, 24, 8, D, B, T, n)
        assert need <= 130 * MB, need / MB


def test_decode_batches_keep_their_pieces():
    """Partial results of a serving batch are small: 64 rows of 24 heads, a piece per 2048 positions."""
    lse = lambda n: -(-64 * 24 * n * 4 // 256) * 256  # noqa: E731
    for span, pieces in ((8003, 4), (65536, 33), (131071, 64)):
        assert qlinear.paged_attention_workspace_size(64, 24, 8, 128, 64, 1, span) == lse(pieces) + 64 * 24 * pieces * 128 * 4
