"""GPU tests of attention over packed sequences at the edges of its sizes."""

import math

import pytest
import torch

from serving_check import cumulative, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("n_q", [[1], [3, 0, 40], [300, 1], [1] * 70])
def test_no_keys_at_all(dtype, D, n_q, monkeypatch):
    """k and v of no rows (which have no memory): every row of a sequence gets 0 and a log-sum-exp of -inf, the others
    stay; natively and through ctypes."""
    from fa2 import _lib
    from fa2.packed import attention_packed
    T, cu = sum(n_q) + 2, cumulative(n_q)
    q, k = randn((T, 8, D), dtype, 1), torch.empty(0, 2, D, dtype=dtype, device="cuda")
    for native in (_lib.native, None):
        monkeypatch.setattr(_lib, "native", native)
        for causal in (True, False):
            out, lse = attention_packed(q, k, k.clone(), cu, torch.zeros_like(cu), causal=causal, return_lse=True,
                                        out=torch.full_like(q, 7.0))
            assert (out[:-2] == 0).all() and (out[-2:] == 7.0).all() and (lse[:, :-2] == -math.inf).all()
            assert (attention_packed(q, k, k, cu, torch.zeros_like(cu), causal=causal)[:-2] == 0).all()
