"""CPU tests of the serving calls' sizes on their way to the C ABI, which takes 32 bits of each."""

import pytest
import torch

from fa2 import _lib
from fa2.paged import KVCache

N = (1 << 32) + 3  # its lower 32 bits alone: 3


def rows(n=3, h=1):
    """[n, h, 16] of any size in the memory of one row"""
    return torch.zeros(1, 1, 16, dtype=torch.float16).expand(n, h, 16)


@pytest.mark.parametrize("q,k", [(rows(N), rows()), (rows(h=N), rows()), (rows(), rows(N)), (rows(), rows(h=N))])
def test_packed_rows_past_32_bits(q, k):
    cu = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="2\\^31"):
        _lib.attn_packed(q, k, k, q, cu, cu, True, 0.1, None, None)


@pytest.mark.parametrize("n", [1 << 31, N])
def test_paged_sizes_past_32_bits(n):
    cu, table = torch.zeros(2, dtype=torch.int32), torch.zeros(1, 4, dtype=torch.int32)
    assert _lib.sequences_of(cu, cu[1:], table, (1 << 31) - 1).n_tokens == (1 << 31) - 1
    with pytest.raises(ValueError, match="tokens"):
        _lib.sequences_of(cu, cu[1:], table, n)
    with pytest.raises(ValueError, match="table_columns"):
        _lib.sequences_of(cu, cu[1:], table[:, :1].expand(1, n), 3)
    with pytest.raises(ValueError, match="sequences"):
        _lib.sequences_of(cu, cu[1:].expand(n), table.expand(n, 4), 3)
    page = torch.zeros(1, 1, 32, 16, dtype=torch.float16)
    for k in (page.expand(n, 1, 32, 16), page.expand(1, n, 32, 16)):
        with pytest.raises(ValueError, match="2\\^31"):
            _lib.cache_of(KVCache(k, k))
    with pytest.raises(ValueError, match="H_q"):
        _lib.attn_paged(rows(h=n), rows(h=n), None, None, True, 0.1, None, None, None)
    with pytest.raises(ValueError, match="H_q"):
        _lib.cache_write(None, None, rows(), rows(), rows(h=n), rows(h=n), None, None)


@pytest.mark.parametrize("shape", [(N, 1, 1), (1, N, 1), (1, 1, N)])
def test_rotary_sizes_past_32_bits(shape):
    x = torch.zeros(1, 1, 1, 16, dtype=torch.float16).expand(*shape, 16)
    positions = torch.zeros(1, 1, dtype=torch.int32).expand(shape[0], shape[2])
    with pytest.raises(ValueError, match="2\\^31"):
        _lib.rotary(x, x, positions, _lib.Rotation(None, 8, 0, 1.0), None)
