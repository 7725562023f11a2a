"""Counts that are no counts, or that the library would take for another one, raise the package's error (CPU only)."""
import pytest
import torch

import coachwhip_amd as cw
from coachwhip_amd import f8, piles

BAD = [0, -1, 2 ** 31, 2 ** 32 + 8, 8 - 2 ** 32, 8.0, "8", None]


@pytest.mark.parametrize("n", BAD)
def test_experts_of_a_sort(n):
    with pytest.raises(cw.CwError, match="experts"):
        piles.sort_picks(torch.zeros(2, 2, dtype=torch.int32), n)


@pytest.mark.parametrize("k", BAD)
def test_codes_of_a_row(k):
    q, scale = torch.zeros(2, 128, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(1, 2)
    for make in (lambda: f8.F8Rows(q, scale, k), lambda: f8.F8Matrix(q, scale, k), lambda: f8.F8ExpertBank(q[None], scale[None], k)):
        with pytest.raises(cw.CwError, match="codes of a row"):
            make()


@pytest.mark.parametrize("k", BAD)
def test_picks_of_a_layer(k):
    with pytest.raises(cw.CwError, match="top_k"):
        f8.F8MoeLayer(None, None, None, top_k=k)


@pytest.mark.parametrize("w", [None, [[1.0]], torch.zeros(2, 3), torch.zeros(2, 3, 4)])
def test_weights_of_a_bank(w):
    with pytest.raises(cw.CwError):
        f8.F8ExpertBank.from_float(w)
