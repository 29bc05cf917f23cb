"""GPU tests of what the serving calls report of lengths, offsets and indices in device memory, and to whom."""
import pytest

from _serving import AMAX, attention64, check, codes, starts

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]
DEV_BAD_INDEX = 13


@pytest.fixture(scope="module")
def torch(pkg):
    import torch
    torch.cuda.set_device(0)
    pkg.device_status()
    return torch


@pytest.fixture(autouse=True)
def clean(pkg):
    yield
    st, words = pkg.device_status()
    assert st == pkg.OK, words


def param(pkg):
    return pkg.FMHAParamI8(*AMAX, 1.0, 1.0)


@pytest.mark.parametrize("max_q", [40, 400])          # a call of chunks, and a batch of single tokens and chunks
def test_a_chunk_on_more_keys_than_waits_are_sized_for_below_a_smaller_bound(pkg, torch, max_q):
    """2^26 + 1 keys where the call says 3000: that sequence is left as it was and reported, the others are computed."""
    D, H, page = 64, 16 if max_q == 400 else 2, 4096
    kc, vc = codes((2, 2, page, D), 1), codes((2, 2, page, D), 2)
    lens_q, lens_k = [40, 1, 33] + [1] * (60 if max_q == 400 else 0), [(1 << 26) + 1, 77, 2999] + [500] * (60 if max_q == 400 else 0)
    table = (torch.arange((1 << 14) + 1, device="cuda") % 2).to(torch.int32)[None].repeat(len(lens_q), 1)
    q = codes((sum(lens_q), H, D), 3)
    o = torch.full((sum(lens_q), H, D), 77.0, dtype=torch.bfloat16, device="cuda")
    pkg.FMHAInferI8Paged(None, param(pkg), pkg.AttnDataDescriptorGrouped(len(lens_q), max_q, 3000, H, 2, D), q, kc, vc, table,
                         torch.tensor(lens_k, dtype=torch.int32, device="cuda"), starts(lens_q), o)
    st, words = pkg.device_status()
    assert st == pkg.ERR_DEVICE and words[0] == DEV_BAD_INDEX and words[2:4] == [0, 0], words
    assert bool((o[:40] == 77.0).all())
    at = 40
    for b in range(1, len(lens_q)):
        n, m = lens_q[b], lens_k[b]
        k, v = (x.transpose(1, 2).reshape(-1, 2, D)[:m] for x in (kc, vc))
        want, scales = attention64(q[at:at + n], k, v, AMAX, True)
        check(o[at:at + n], want, scales, m, "bf16", AMAX, 1.0, max_q * H // 2, f"sequence {b}", own=n * H // 2)
        at += n
