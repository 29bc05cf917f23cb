"""GPU tests of batches of thousands of sequences in which few bring many tokens: their units are found without going through all the others for each."""
import pytest

from _serving import AMAX, attention64, check, codes, starts

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


@pytest.fixture(scope="module")
def torch(pkg):
    import torch
    torch.cuda.set_device(0)
    pkg.device_status()
    return torch


def batch(pkg, torch, B, long, H, Hkv, D, page=64, keys=70):
    """(call, output, check of some sequences): sequences of one token on `keys` keys, those in `long` {index: tokens} on as many keys as tokens."""
    lens_q, lens_k = [long.get(b, 1) for b in range(B)], [long.get(b, keys) for b in range(B)]
    pages = -(-max(lens_k) // page)
    kc, vc = codes((pages, Hkv, page, D), 1), codes((pages, Hkv, page, D), 2)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].repeat(B, 1)          # all sequences on the same keys
    q, cu = codes((sum(lens_q), H, D), 3), starts(lens_q)
    o = torch.full((sum(lens_q), H, D), 77.0, dtype=torch.bfloat16, device="cuda")
    args = (None, pkg.FMHAParamI8(*AMAX, 1.0, 1.0), pkg.AttnDataDescriptorGrouped(B, max(lens_q), max(lens_k), H, Hkv, D), q, kc, vc, table,
            torch.tensor(lens_k, dtype=torch.int32, device="cuda"), cu, o)

    def verify(which):
        for b in which:
            n, m, at = lens_q[b], lens_k[b], int(cu[b])
            k, v = (x.transpose(1, 2).reshape(-1, Hkv, D)[:m] for x in (kc, vc))
            want, scales = attention64(q[at:at + n], k, v, AMAX, True)
            check(o[at:at + n], want, scales, m, "bf16", AMAX, 1.0, max(lens_q) * H // Hkv, f"sequence {b}", own=n * H // Hkv)
        assert not bool((o == 77.0).all(-1).any()), "rows that nobody wrote"
    return (lambda: pkg.FMHAInferI8Paged(*args)), o, verify


@pytest.mark.parametrize("B,long", [(2100, {2099: 900}), (2100, {0: 700, 2000: 33, 2099: 129}), (1500, {700: 500, 701: 90, 733: 64, 40: 300}),
                                    (1000, {b: 20 + (7 * b) % 60 for b in range(300, 700, 3)}), (33, {32: 400})])
@pytest.mark.parametrize("H,Hkv,D", [(8, 2, 64), (4, 4, 128)])
def test_few_long_sequences_among_many(pkg, torch, B, long, H, Hkv, D):
    call, o, verify = batch(pkg, torch, B, long, H, Hkv, D)
    call()
    verify(sorted(set(list(long) + [0, 1, 31, 32, B // 2, B - 2, B - 1])))
    assert pkg.device_status()[0] == pkg.OK


def test_a_long_sequence_does_not_pay_for_thousands_of_others(pkg, torch):
    """8192 tokens among 4096 sequences take no more than four times as long as among two.  (Eleven times, while all sequences were looked at for every level of pairs; twice now.)"""
    times = []
    for B in (2, 4096):
        call, o, verify = batch(pkg, torch, B, {B - 1: 8192}, 32, 8, 128)
        best = []
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            call()
            b.record()
            torch.cuda.synchronize()
            best.append(a.elapsed_time(b))
        times.append(min(best))
    assert times[1] < 4 * times[0], times
    assert pkg.device_status()[0] == pkg.OK
