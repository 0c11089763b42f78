"""The comparison of tests/_bias_sums.py on the host: it holds for a sum in 32 bits, a lost part is seen."""

import pytest
import torch

from tests import _bias_sums as S


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_lost_part_is_seen(dtype):
    terms = torch.randn((4096, 64, 24), generator=torch.Generator().manual_seed(0))     # parts of 64 terms
    parts = terms.sum(1)
    flat = terms.flatten(0, 1)
    additions = S.depth(4096, 64, 8)
    S.check(parts.sum(0).to(dtype), flat, additions, 4096 * 64 // 8)
    for k in (0, 3, 7):     # what one of eight CTAs brings
        kept = torch.cat((parts[:512 * k], parts[512 * (k + 1):]))
        with pytest.raises(AssertionError):
            S.check(kept.sum(0).to(dtype), flat, additions)
    with pytest.raises(AssertionError):
        S.check(torch.zeros(24, dtype=dtype), flat, additions)
    with pytest.raises(AssertionError):
        S.check(parts.sum(0).to(dtype), flat, 2 ** 24, 4096 * 64 // 8)      # a limit that could not see it
