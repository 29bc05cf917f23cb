"""GPU tests of the quantiser next to the borders of its codes: the product is rounded to fp32 before one half is added and the sum rounded again, as the
oracle does, which a fused multiply-add would not."""
import numpy as np
import pytest

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]
SWEEP = 148 * 8 * 1024


def borders(amax):
    """Numbers next to half a step whose code depends on that rounding."""
    scale, found = np.float32(127.0) / amax, []
    for half in (0.5, -0.5):
        x = np.float32(half) / scale
        for _ in range(4):
            x = np.nextafter(x, np.float32(-np.inf))
        for _ in range(8):
            rounded = np.float32(np.float32(x * scale) + np.float32(0.5))
            if np.floor(rounded) != np.floor(np.float32(np.float64(x) * np.float64(scale) + 0.5)):
                found.append(x)
            x = np.nextafter(x, np.float32(np.inf))
    return found


@pytest.mark.parametrize("n", [67, 4099, 262144, 300007, 524289, 3 * SWEEP + 5, 20 * SWEEP + 3])
def test_the_product_is_rounded_before_the_sum(pkg, oracle, n):
    import torch
    rng = np.random.default_rng(n)
    tried = 0
    while tried < (40 if n < 10000 else 4):
        amax = np.float32(rng.uniform(0.1, 60.0))
        found = borders(amax)
        if not found:
            continue
        tried += 1
        x = (rng.standard_normal(n, dtype=np.float32) * (amax / 8)).clip(-amax, amax)
        at = rng.permutation(n)[: max(len(found) * 2, n // 1000 + 64)]
        x[at] = np.resize(np.array(found, np.float32), at.size)
        x[at[-1]] = amax
        out, got = torch.empty(n, dtype=torch.int8, device="cuda"), torch.zeros(1, device="cuda")
        pkg.quantize_f32(None, torch.from_numpy(x).cuda(), out, got)
        assert np.float32(got.item()) == amax
        off = np.flatnonzero(out.cpu().numpy() != oracle.quantize(x, float(amax)))
        assert off.size == 0, f"range {float(amax).hex()}: {off.size} codes off, the first for {float(x[off[0]]).hex()}"
    assert pkg.device_status()[0] == pkg.OK
