"""The 8-bit operators and the AdamW step at the ends of the numbers' range: moments that overflow."""
import numpy as np
import pytest
import torch

import blocks_reference as R

pytestmark = pytest.mark.gpu
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def raw(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t.view(torch.int32 if t.element_size() == 4 else torch.int16)


# ----------------------------------------------------------------------------------------------------------------- AdamW
@pytest.mark.parametrize("value", [1e21, -1e21, float("inf"), float("nan")])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_gradient_without_a_square_stays_with_its_element(bits, value):
    """One gradient whose square is over float32's largest number, or that is no number: every other element of its block of 128 moves, bit for bit,
    as it does with a zero in that place, in this step and in the ones behind it.  A finite one leaves the weight finite, which only
    decays then."""
    import sd_mecha_amd as amd
    n, at, steps = 384, 128 + 17, 4
    seg = torch.tensor([[0, n]], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    p0, grads = torch.randn(n, device="cuda", generator=g) * 0.02, torch.randn(steps, n, device="cuda", generator=g) * 1e-3
    grads[:, at] = 0.0
    runs = []
    for bad in (False, True):
        st, p, flags = amd.adamw_state(n, "cuda", bits), p0.clone(), torch.zeros(1, dtype=torch.int32, device="cuda")
        trace = []
        for t in range(1, steps + 1):
            x = grads[t - 1].clone()
            if bad and t == 1:
                x[at] = value
            amd.adamw_step(p, x, segments=seg, step=t, lr=1e-2, weight_decay=0.1, seed=3, flags=flags, **st)
            trace.append([p.clone()] + [v.clone() for v in st.values()] + [int(flags)])
            flags.zero_()
        runs.append(trace)
    others = torch.arange(n, device="cuda") != at
    for t, (clean, bad) in enumerate(zip(*runs)):
        for x, y in zip(clean[:-1], bad[:-1]):
            same = raw(x) == raw(y)
            assert bool(same[others].all() if same.numel() == n else same.all()), t
        assert clean[-1] == 0
        if np.isfinite(value):
            assert float(bad[0][at]) == float(clean[0][at]) and bad[-1] == 2          # the gradient is finite, its square is not
        else:
            assert bool(bad[0][at].isnan()) and bad[-1] & 2 and bad[-1] & 1
        if bits == 8:
            assert bool(bad[2][at].float().isnan()) and bool(bad[1][at].float().isnan()) == (not np.isfinite(value))
    # and the others do move: weights in every step, roots over the steps
    assert bool((runs[1][0][0] != p0)[others].all()) and all(bool((runs[1][t][0] != runs[1][t - 1][0])[others].all()) for t in range(1, steps))
