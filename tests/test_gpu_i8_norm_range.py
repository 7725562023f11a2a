"""RMS norms whose values leave f32: a scale is finite and so are its row's values, or it is NaN and the codes are zero."""
import pytest
import torch

from coachwhip_amd import i8

from .test_gpu_i8 import U, codes_of, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", [2, 700, 32768])
def test_norm_of_values_beyond_f32(k):
    """One value a row: the norm is weight * sqrt(k) there (eps 0), up to 181 times f32's largest, and the scale that over 127."""
    say("norm beyond f32", k)
    top = torch.finfo(torch.float32).max
    weights = torch.tensor([1.0, top / 256, top / 127, top / 2, 0.69 * top, 0.75 * top, top], dtype=torch.float64)
    for w in weights.tolist():
        x = torch.zeros(3, k, device="cuda")
        x[0, k - 1], x[1, 0], x[2, :] = 2.0, -0.5, 1.0
        r, _, y = i8.rmsnorm_i8(x, torch.full((k,), w, device="cuda"), 0.0, keep_y=True)
        wf = float(torch.tensor(w, dtype=torch.float32))
        for row, (at, want) in enumerate(((k - 1, wf * k ** 0.5), (0, -wf * k ** 0.5), (0, wf))):
            scale, code = float(r.scale[row]), float(codes_of(r)[row, at])
            if abs(want) / 127 <= top:
                assert abs(scale - abs(want) / 127) <= (U + 1e-13) * abs(want) / 127 and code == (127 if want > 0 else -127)
                if row < 2:
                    assert torch.count_nonzero(r.q[row]) == 1
            else:
                assert scale != scale and not r.q[row].any()
