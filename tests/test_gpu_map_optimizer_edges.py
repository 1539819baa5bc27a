"""-m gpu : gs_localization_amd.map_optimizer where values, options and calls meet that tests/test_gpu_map_optimizer.py takes apart: roots that
overflow, betas that change, several groups, layouts that torch has not resolved yet, codes that an eviction raises."""
import copy
import math
import pickle

import numpy as np
import pytest
import torch

from oracle import map_optimizer_oracle as O
from tests.test_gpu_map_optimizer import DEV, E, HALF, MO, SIZES, Guarded, bound32, check8, clocks, n64, random_codes, small_map

pytestmark = pytest.mark.gpu


def codes(n):
    return torch.zeros(n, dtype=torch.uint8, device=DEV), torch.zeros(n, dtype=torch.int8, device=DEV), torch.zeros((n + 255) // 256, dtype=torch.uint8, device=DEV)


# ---- 8-bit moments: values at the ends ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("beside", [0.0, 1e-5, 1.0])
def test_overflowed_root_keeps_the_momentums_sign(dtype, shift, beside):
    """One gradient per block of 256 whose square is no float: its root's code is 255 and |exp_avg| is more than the span times what that code
    stands for (1e19 and more against 2 roots of the largest neighbour), so its ratio is 127 with the gradient's sign.  The
    neighbours round as if it were not there, and the next step does not go up the gradient."""
    bad = [3e38, -3e38, 1e30, -1e30, 1e20, -1e20, float("inf"), -float("inf"), 2e38]
    n = 2048 + 100          # eight blocks of whole waves, one of a partial wave
    gen = torch.Generator(device=DEV).manual_seed(50)
    g = torch.randn(n, generator=gen, device=DEV) * beside
    at = torch.arange(len(bad), device=DEV) * 256 + 17
    out = []
    for values in (bad, [0.0] * len(bad)):
        gg = g.clone()
        gg[at] = torch.tensor(values, device=DEV)
        p, gg = Guarded(torch.ones(n, device=DEV), shift), Guarded(gg.to(dtype), shift)
        rms, ratio, window = (Guarded(x, shift) for x in codes(n))
        ck = clocks(1, 0, (0.9, 0.999))
        step = lambda: MO().adamw_step_8bit([p.t], [gg.t], [rms.t], [ratio.t], [window.t], ck, lr=0.1, seed=3)          # noqa: E731
        step()
        out.append([x.t.clone() for x in (p, rms, ratio, window)])
    (p1, rms1, ratio1, window1), (p0, rms0, ratio0, window0) = out
    sign = torch.tensor([math.copysign(1.0, x) for x in bad], device=DEV)
    assert ratio1[at].tolist() == (127 * sign).tolist()
    assert (rms1[at] == 255).all()
    finite = torch.tensor([math.isfinite(x) for x in bad], device=DEV)
    assert (p1[at][finite] == 1.0).all() and p1[at][~finite].isnan().all()          # (finite / infinite is nothing, infinite / infinite is NaN)
    others = torch.ones(n, dtype=torch.bool, device=DEV)
    others[at] = False
    for x, y in ((p1, p0), (rms1, rms0), (ratio1, ratio0)):
        assert torch.equal(x[others], y[others])
    assert torch.equal(window1, window0)
    q = torch.ones(n, device=DEV)
    MO().adamw_step_8bit([q], [torch.zeros(n, device=DEV)], [rms1], [ratio1], [window1], clocks(1, 1, (0.9, 0.999)), lr=0.1, seed=3)
    assert ((q[at] - 1.0) * sign <= 0).all()


@pytest.mark.parametrize("eps", [1e30, 2.0 ** 100, 1e35, 2.0 ** 127, 3e38, math.inf])
def test_first_8_bit_step_with_a_large_eps(eps):
    """The same bits as with 32-bit moments (nothing has been rounded to a byte yet), whatever eps is added to the root."""
    n = 4096
    gen = torch.Generator(device=DEV).manual_seed(51)
    g = torch.randn(n, generator=gen, device=DEV) * torch.exp2(torch.randint(-55, 60, (n,), generator=gen, device=DEV).float())
    p = torch.randn(n, generator=gen, device=DEV)
    q = p.clone()
    a = codes(n)
    MO().adamw_step([p], [g], [torch.zeros_like(p)], [torch.zeros_like(p)], clocks(1, 0, (0.9, 0.999)), lr=1e25, eps=eps)
    MO().adamw_step_8bit([q], [g], [a[0]], [a[1]], [a[2]], clocks(1, 0, (0.9, 0.999)), lr=1e25, eps=eps)
    assert bool(p.isfinite().all()) and torch.equal(p.view(torch.int32), q.view(torch.int32))
