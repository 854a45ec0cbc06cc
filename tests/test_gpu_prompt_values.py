"""Values that are no numbers in prompts without a mask: every query of their sequence gets them, wherever they lie."""
import pytest
import torch

from tests.test_gpu_prompt import DT, _inputs

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.mark.parametrize("lens,at", [([40], 0), ([40], 33), ([200, 90], 195), ([200, 90], 130), ([90, 200], 85), ([2100, 1], 2090), ([129], 128)])
@pytest.mark.parametrize("H,D,Dv,dt", [(2, 64, 64, "fp16"), (2, 128, 128, "bf16"), (128, 192, 128, "bf16"), (2, 256, 256, "fp16"), (2, 72, 40, "bf16")])
@pytest.mark.parametrize("bad", [INF, -INF, float("nan")])
def test_without_a_mask_all_queries_see_them(dev, lens, at, H, D, Dv, dt, bad):
    from arcagi2_flashnext_dots3_amd import kernels
    q, k, v, start = _inputs(lens, H, H // 2, D, Dv, DT[dt], D + at)
    args = [x.to(dev) for x in (q, k, v, start)] + [0.3 * D ** -0.5]
    want, wl = kernels.attend_prompt(*args, causal=False)
    args[2][at, 0, Dv - 3] = bad
    out, lse = kernels.attend_prompt(*args, causal=False)
    torch.cuda.synchronize()
    b = 0 if at < lens[0] else 1
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[int(start[b]):int(start[b + 1]), :2, Dv - 3] = True
    assert bool((out[hit].isnan() if bad != bad else out[hit] == bad).all())
    assert torch.equal(out[~hit], want[~hit]) and torch.equal(lse, wl)


def test_infinities_of_both_signs(dev):
    """One of each in the last tile: no number for any query; under a mask the sign of the first until the second is seen."""
    from arcagi2_flashnext_dots3_amd import kernels
    q, k, v, start = _inputs([100], 2, 1, 128, 128, torch.bfloat16, 1)
    v[70, 0, 9], v[90, 0, 9] = INF, -INF
    args = [x.to(dev) for x in (q, k, v, start)] + [0.03]
    full, masked = (kernels.attend_prompt(*args, causal=c)[0][:, :, 9].float() for c in (False, True))
    torch.cuda.synchronize()
    assert bool(full.isnan().all())
    assert bool(masked[:70].isfinite().all()) and bool((masked[70:90] == INF).all()) and bool(masked[90:].isnan().all())
