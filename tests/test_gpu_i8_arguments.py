"""Arguments of the 8-bit integer path that are missing or of another kind: an error of the package, before any launch."""
import pytest
import torch

import coachwhip_amd as cw
from coachwhip_amd import formats as F
from coachwhip_amd import i8, ops

pytestmark = pytest.mark.gpu


def test_norm_without_a_weight():
    x = torch.ones(2, 128, device="cuda")
    for weight in (None, [1.0] * 128, torch.ones(128), torch.ones(128, device="cuda").half(), torch.ones(128, 2, device="cuda")[:, 0]):
        with pytest.raises(cw.CwError):
            i8.rmsnorm_i8(x, weight, 1e-6)


def test_banks_in_row_groups_are_refused():
    """(GGUF rows are: the dequantizer takes them)"""
    raw = torch.zeros(2 * 16 * 4 * 17, dtype=torch.uint8, device="cuda")
    bank = ops.ExpertBank(raw, F.MXFP4, 16, 128, 2, 16 * 4 * 17)
    assert i8.I8ExpertBank.from_bank(bank).q.shape == (2, 16, 128)
    with pytest.raises(cw.CwError):
        i8.I8ExpertBank.from_bank(bank.rows16())
