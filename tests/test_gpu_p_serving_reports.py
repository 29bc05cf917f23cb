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


def small_forward(pkg, torch):
    """A padded forward call: what it gives, as a function, and the arguments."""
    q, k, v = (codes((1, 2, 128, 64), s) for s in (11, 12, 13))
    mask = torch.zeros((1, 128), dtype=torch.int8, device="cuda")
    return lambda o, check=True: pkg.FMHAInferI8(None, pkg.FMHAParamI8(*AMAX, 1.0, 1.0), pkg.AttnDataDescriptor(1, 128, 2, 64), q, k, v, mask, o, True, check=check)


def bad_calls(pkg, torch):
    """A page, a length, an offset and a slot that point outside their tensors, one call each: its code and the detail that is reported."""
    kc, vc = codes((4, 1, 16, 64), 1), codes((4, 1, 16, 64), 2)
    q, o = codes((2, 1, 64), 3), torch.empty((2, 1, 64), dtype=torch.bfloat16, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    desc = pkg.AttnDataDescriptorGrouped(2, 1, 32, 1, 1, 64)
    x = torch.zeros((2, 1, 64), device="cuda")
    codes_out = codes((2, 1, 64), 4)
    return [(lambda: pkg.FMHAInferI8Paged(None, param(pkg), desc, q, kc, vc, i32(0, 9, 1, 2).view(2, 2), i32(20, 20), starts([1, 1]), o), 1, 0),
            (lambda: pkg.FMHAInferI8Paged(None, param(pkg), desc, q, kc, vc, i32(0, 3, 1, 2).view(2, 2), i32(20, 33), starts([1, 1]), o), 0, 1),
            (lambda: pkg.FMHAInferI8Packed(None, param(pkg), desc, q, q, q, i32(0, 1, 3), i32(0, 1, 2), o), 0, 1),
            (lambda: pkg.rope_quantize_append(None, param(pkg), x, x, x, i32(0, 0), None, codes_out, kc, vc, slots=torch.tensor([0, 64], device="cuda")), 2, 1)]


def test_an_index_outside_is_nobody_elses_error(pkg, torch):
    """It is reported through the status words alone: the next calls run, whoever makes them."""
    forward = small_forward(pkg, torch)
    want = torch.empty((1, 2, 128, 64), dtype=torch.int8, device="cuda")
    forward(want)
    for call, detail, which in bad_calls(pkg, torch):
        call()
        torch.cuda.synchronize()
        o = torch.zeros_like(want)
        forward(o)
        assert torch.equal(o, want)
        q, k, v = codes((5, 2, 64), 1), codes((5, 2, 64), 2), codes((5, 2, 64), 3)
        got = torch.empty((5, 2, 64), dtype=torch.bfloat16, device="cuda")
        cu = starts([5])
        pkg.FMHAInferI8Packed(None, param(pkg), pkg.AttnDataDescriptorGrouped(1, 5, 5, 2, 2, 64), q, k, v, cu, cu, got)
        exact, scales = attention64(q, k, v, AMAX, True)
        check(got, exact, scales, 5, "bf16", AMAX, 1.0, 5)
        st, words = pkg.device_status()
        assert st == pkg.ERR_DEVICE and words[0] == DEV_BAD_INDEX and words[2:4] == [detail, which], words
        assert pkg.device_status()[0] == pkg.OK


def test_an_index_outside_hides_no_wait_that_ran_out(pkg, torch):
    forward = small_forward(pkg, torch)
    o = torch.empty((1, 2, 128, 64), dtype=torch.int8, device="cuda")
    forward(o)
    call, detail, which = bad_calls(pkg, torch)[0]
    call()
    torch.cuda.synchronize()
    pkg.debug_wait_probe(None, 4_000_000)                 # a kernel that waits two milliseconds for nothing
    torch.cuda.synchronize()
    forward(o, check=False)
    assert pkg.lib().fmha_i8_sm100_last_status() == pkg.ERR_DEVICE
    st, words = pkg.device_status()
    assert st == pkg.ERR_DEVICE and words[0] == 10 and words[4] == DEV_BAD_INDEX and words[6:8] == [detail, which], words
    forward(o)


@pytest.mark.parametrize("D,H", [(64, 4), (128, 48)])
def test_tokens_where_the_call_allows_none_are_reported(pkg, torch, D, H):
    """max_seq_q = 0 with tokens on the device: they may be left as they were, but not without a word.  Without tokens there is nothing to say."""
    q, k = codes((5, H, D), 1), codes((5, 2, D), 2)
    o = torch.full((5, H, D), 7.0, dtype=torch.bfloat16, device="cuda")
    desc = pkg.AttnDataDescriptorGrouped(2, 0, 5, H, 2, D)
    lens, table = torch.tensor([3, 2], dtype=torch.int32, device="cuda"), torch.zeros((2, 1), dtype=torch.int32, device="cuda")
    kc = codes((1, 2, 16, D), 3)
    for tokens in (starts([0, 3]), starts([3, 2]), starts([0, 0])):
        for call in (lambda: pkg.FMHAInferI8Packed(None, param(pkg), desc, q, k, k, tokens, starts([2, 3]), o),
                     lambda: pkg.FMHAInferI8Paged(None, param(pkg), desc, q, kc, kc, table, lens, tokens, o)):
            call()
            st, words = pkg.device_status()
            if int(tokens[-1]) == 0:
                assert st == pkg.OK and bool((o == 7.0).all())
            else:
                assert st == pkg.ERR_DEVICE and words[0] == DEV_BAD_INDEX and words[2] == 0, words
            o.fill_(7.0)


@pytest.mark.parametrize("page", [0, 16])
def test_without_a_rotation_any_position_will_do(pkg, torch, page):
    """No table, no positions to look up: tokens with positions below zero and far out are quantised and stored like the others, and nothing is reported."""
    T, H, Hkv, D = 6, 3, 1, 64
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    q, k, v = (torch.randn((T, h, D), device="cuda", generator=g).bfloat16() for h in (H, Hkv, Hkv))
    outs = []
    for positions in ([0, 1, 2, 3, 4, 5], [-1, 2 ** 31 - 1, -2 ** 31, 7, -5, 0]):
        q_out = torch.zeros((T, H, D), dtype=torch.int8, device="cuda")
        ko, vo = (torch.zeros((1, Hkv, page, D) if page else (T, Hkv, D), dtype=torch.int8, device="cuda") for _ in range(2))
        pkg.rope_quantize_append(None, param(pkg), q, k, v, torch.tensor(positions, dtype=torch.int32, device="cuda"), None, q_out, ko, vo,
                                 slots=torch.arange(T, device="cuda") if page else None)
        outs.append((q_out, ko, vo))
        st, words = pkg.device_status()
        assert st == pkg.OK, words
    assert all(torch.equal(a, b) for a, b in zip(*outs)) and bool(outs[0][1].any())
