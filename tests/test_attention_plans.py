"""CPU: the workspace that paged attention asks for (a query of sizes, no GPU call)."""
import pytest

import qlinear
from qlinear import _lib
from test_decoder import _attention

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


def test_long_chunks_are_refused_only_where_a_grid_ends():
    """scale=-1 is refused after the sizes: a call that gets there has sizes that can run."""
    call = lambda **kw: _attention(_lib.lib(), **{**dict(scale=-1.0, pst=1 << 40, P=1 << 20, tst=1 << 20), **kw})  # noqa: E731
    for D in (64, 96, 128, 256):
        for Hq, Hkv in ((24, 8), (16, 1), (8, 8)):
            n = 1 << 20
            assert call(T=n, mq=n, mk=n, Hq=Hq, Hkv=Hkv, D=D) == (_lib.QL_EUNSUPPORTED if D in (64, 128) and Hq == 16 else _lib.QL_EINVAL_ARG)
            n = 65535 * 256 * Hkv // Hq  # rows of a kv head in 65535 tiles of 256
            assert call(T=n, mq=n, mk=n, Hq=Hq, Hkv=Hkv, D=D) == _lib.QL_EINVAL_ARG
    n = 65535 * 256 + 1
    assert call(T=n, mq=n, mk=n, Hq=4, Hkv=4, D=128) == _lib.QL_EUNSUPPORTED and call(T=n, mq=n, mk=n, Hq=4, Hkv=4, D=96) == _lib.QL_EINVAL_ARG
    n = (1 << 30) + 1
    assert call(T=n, mq=n, mk=100, Hq=4, Hkv=4, D=96) == _lib.QL_EUNSUPPORTED


def test_any_sizes_have_an_answer():
    """No new tokens, nothing cached, bounds at their ends: the query returns."""
    ask = qlinear.paged_attention_workspace_size
    for D in (64, 96, 128, 256):
        for max_q in (0, 1, 41):
            for max_kv in (0, 1, 300, 7000, 1 << 30):
                for B in (0, 1, 2, 40):
                    assert ask(41, 6, 2, D, B, max_q, max_kv) >= 0 and ask(41, 6, 2, D, B, max_q, max_kv, 64) >= 0
