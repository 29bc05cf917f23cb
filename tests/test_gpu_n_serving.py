"""GPU tests of the serving calls -- rope_table, rope_quantize_append, FMHAInferI8Packed, FMHAInferI8Paged -- against their definitions in 64
bits.  Codes have to be equal; outputs stay within the roundings counted in _serving.tolerance()."""
import math

import pytest

from _serving import AMAX, TYPES, assert_same, attention64, check, codes, quantise64, rotate64, starts

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(600)]
O_AMAX = 2.5
FILL = {"int8": 0x5A, "bf16": 77.0, "fp16": 77.0}


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
    return pkg.FMHAParamI8(*AMAX, O_AMAX, 1.0)


# ------------------------------------------------------------------------------------------------ rotary positions, append

def inv_freq_of(torch, rot, base=10000.0):
    return torch.tensor([base ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device="cuda")


def make_table(pkg, torch, rot, positions, magnitude=1.0):
    freq = inv_freq_of(torch, rot)
    table = torch.empty((2, positions, rot), dtype=torch.float32, device="cuda")
    pkg.rope_table(None, freq, table, magnitude)
    return freq, table


@pytest.mark.parametrize("rot,positions,magnitude", [(16, 1, 1.0), (64, 1000, 1.0), (128, 200001, 1.25), (96, 77, 0.5)])
def test_rope_table(pkg, torch, rot, positions, magnitude):
    freq, table = make_table(pkg, torch, rot, positions, magnitude)
    angle = torch.arange(positions, device="cuda").double()[:, None] * freq
    want = torch.stack((torch.cos(angle), torch.sin(angle)), -1).flatten(1) * magnitude
    # 48 bits in the two planes, a 64-bit sine or cosine (2 steps of 2^-53), a product
    assert float((table.double().sum(0) - want).abs().max()) <= magnitude * (2.0 ** -48 + 4 * 2.0 ** -53)
    assert float((table[0].double() - want).abs().max()) <= magnitude * 2.0 ** -24


def make_qkv(torch, T, H, Hkv, D, dtype, seed, fused=True):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if fused:
        x = torch.randn((T, H + 2 * Hkv, D), generator=g, device="cuda").to(TYPES[dtype])
        return x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    return tuple(torch.randn((T, h, D), generator=g, device="cuda").to(TYPES[dtype]) for h in (H, Hkv, Hkv))


APPEND = [
    # T, H, Hkv, D, rot, interleaved, dtype, page (0: packed), fused
    (1, 1, 1, 64, 64, False, "bf16", 16, True),
    (1, 12, 12, 64, 0, False, "fp32", 16, False),
    (3, 7, 1, 128, 128, True, "fp16", 32, True),
    (17, 28, 4, 128, 64, False, "bf16", 128, True),
    (65, 5, 5, 64, 16, True, "bf16", 64, False),
    (130, 32, 8, 128, 128, False, "fp32", 16, True),
    (1000, 6, 2, 64, 32, False, "fp16", 0, True),
    (777, 16, 2, 128, 96, True, "bf16", 0, False),
    (5000, 9, 3, 128, 128, False, "bf16", 256, True),
]


@pytest.mark.parametrize("T,H,Hkv,D,rot,interleaved,dtype,page,fused", APPEND)
def test_append_gives_the_exact_codes(pkg, torch, T, H, Hkv, D, rot, interleaved, dtype, page, fused):
    freq, table = make_table(pkg, torch, rot, 3 * T + 100000, 1.1) if rot else (torch.empty(0, dtype=torch.float64, device="cuda"), None)
    q, k, v = make_qkv(torch, T, H, Hkv, D, dtype, T + rot, fused)
    g = torch.Generator(device="cuda")
    g.manual_seed(T)
    pos = torch.randint(0, 3 * T + 100000, (T,), dtype=torch.int32, device="cuda", generator=g)
    q_out = torch.full((T + 1, H, D), 0x5A, dtype=torch.int8, device="cuda")
    want_q, want_k = (quantise64(rotate64(x.double(), pos, freq, 1.1, interleaved), a) for x, a in ((q, AMAX[0]), (k, AMAX[1])))
    want_v = quantise64(v.double(), AMAX[2])
    if page:
        pages = -(-T // page) + 2
        # K and V of a page side by side: the pages are twice as far apart as they are long
        both = torch.full((pages, 2, Hkv, page, D), 0x5A, dtype=torch.int8, device="cuda")
        kc, vc = both[:, 0], both[:, 1]
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:T].contiguous()
        if T > 2:
            slots[1] = -1
        pkg.rope_quantize_append(None, param(pkg), q, k, v, pos, table, q_out[:T], kc, vc, slots=slots, interleaved=interleaved)
        want = both.new_full((2, pages * page, Hkv, D), 0x5A)
        kept = slots >= 0
        want[0, slots[kept]], want[1, slots[kept]] = want_k[kept], want_v[kept]
        assert_same(kc.transpose(1, 2).reshape(-1, Hkv, D), want[0])
        assert_same(vc.transpose(1, 2).reshape(-1, Hkv, D), want[1])
    else:
        ko, vo = (torch.full((T + 1, Hkv, D), 0x5A, dtype=torch.int8, device="cuda") for _ in range(2))
        pkg.rope_quantize_append(None, param(pkg), q, k, v, pos, table, q_out[:T], ko[:T], vo[:T], interleaved=interleaved)
        assert_same(ko[:T], want_k)
        assert_same(vo[:T], want_v)
        assert bool((ko[T] == 0x5A).all()) and bool((vo[T] == 0x5A).all())
    assert_same(q_out[:T], want_q)
    assert bool((q_out[T] == 0x5A).all())


def test_append_decides_ties_and_takes_what_is_no_number(pkg, torch):
    """Values exactly on a border between two codes go up, at any sign; beyond the range they saturate; not a number gives 0."""
    amax = 127.0 / 32.0                                           # a code is 1/32: every multiple of 1/64 is a border or a code
    p = pkg.FMHAParamI8(amax, amax, amax, 1.0, 1.0)
    x = (torch.arange(-320, 320, device="cuda").float() / 64.0).view(-1, 1, 64)
    tail = torch.zeros((1, 1, 64), device="cuda")
    tail[0, 0, :8] = torch.tensor([math.inf, -math.inf, math.nan, 3e38, -3e38, 1e-45, -1e-45, 0.5 / 32], device="cuda")
    x = torch.cat((x, tail)).contiguous()
    T = x.shape[0]
    out = [torch.empty((T, 1, 64), dtype=torch.int8, device="cuda") for _ in range(3)]
    pkg.rope_quantize_append(None, p, x, x, x, torch.zeros(T, dtype=torch.int32, device="cuda"), None, *out)
    for o in out:
        assert_same(o, quantise64(x.double(), amax))
    # turned by nothing: position 0 of a table is the identity, and a product with infinity that has no value gives 0
    _, table = make_table(pkg, torch, 64, 4)
    pkg.rope_quantize_append(None, p, x, x, x, torch.zeros(T, dtype=torch.int32, device="cuda"), table, *out)
    want = quantise64(rotate64(x.double(), torch.zeros(T, device="cuda"), inv_freq_of(torch, 64), 1.0, False), amax)
    assert_same(out[0], want)
    assert_same(out[1], want)
    assert_same(out[2], quantise64(x.double(), amax))


def test_append_reports_positions_and_slots_outside(pkg, torch):
    q, k, v = make_qkv(torch, 4, 2, 1, 64, "bf16", 1)
    freq, table = make_table(pkg, torch, 64, 10)
    kc, vc = (torch.zeros((2, 1, 16, 64), dtype=torch.int8, device="cuda") for _ in range(2))
    q_out = torch.zeros((4, 2, 64), dtype=torch.int8, device="cuda")
    for pos, slots, missing_q in (([0, 1, 10, 3], [0, 1, 2, 3], [2]), ([0, -1, 2, 3], [0, 1, 2, 3], [1]), ([0, 1, 2, 3], [0, 32, 2, 3], [])):
        q_out.zero_(); kc.zero_(); vc.zero_()
        pkg.rope_quantize_append(None, param(pkg), q, k, v, torch.tensor(pos, dtype=torch.int32, device="cuda"), table, q_out, kc, vc,
                                 slots=torch.tensor(slots, device="cuda"))
        st, words = pkg.device_status()
        assert st == pkg.ERR_DEVICE and words[0] == 13 and words[2] == 2
        ok = [t for t in range(4) if 0 <= pos[t] < 10]
        want = quantise64(rotate64(q[ok].double(), torch.tensor(pos, device="cuda")[ok], freq, 1.0, False), AMAX[0])
        assert_same(q_out[ok], want)
        assert not bool(q_out[missing_q].any())
        stored = [t for t in ok if 0 <= slots[t] < 32]
        flat = vc.transpose(1, 2).reshape(-1, 64)
        assert_same(flat[[slots[t] for t in stored]], quantise64(v[stored].double(), AMAX[2])[:, 0])
        assert int((flat != 0).any(-1).sum()) == len(stored)


# ------------------------------------------------------------------------------------------------ packed prompts

def run_packed(pkg, torch, lens_q, lens_k, H, Hkv, D, causal, out, seed, tail=3, max_q=None, max_k=None, fused=False, stream=None):
    same = lens_k is None
    lens_k = lens_q if same else lens_k
    tq, tk = sum(lens_q) + tail, sum(lens_k) + (tail if same else 0)
    if fused and same:
        x = codes((tq, H + 2 * Hkv, D), seed)
        q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    else:
        q, k, v = codes((tq, H, D), seed), codes((tk, Hkv, D), seed + 1), codes((tk, Hkv, D), seed + 2)
    o = torch.full((tq, H, D), FILL[out], dtype=TYPES[out], device="cuda")
    cu_q, cu_k = starts(lens_q), starts(lens_k)
    desc = pkg.AttnDataDescriptorGrouped(len(lens_q), max_q or max(lens_q), max(lens_k) if max_k is None else max_k, H, Hkv, D)
    pkg.FMHAInferI8Packed(stream, param(pkg), desc, q, k, v, cu_q, cu_q if same else cu_k, o, causal=causal)
    at_q = at_k = 0
    for n, m in zip(lens_q, lens_k):
        want, spread = attention64(q[at_q:at_q + n], k[at_k:at_k + m], v[at_k:at_k + m], AMAX, causal)
        check(o[at_q:at_q + n], want, spread, m, out, AMAX, O_AMAX, desc.max_seq_q * H // Hkv, f"{n} tokens on {m} keys", own=n * H // Hkv)
        at_q += n
        at_k += m
    assert bool((o[at_q:] == FILL[out]).all()), "tokens behind the last sequence were touched"
    return q, k, v, o


PACKED = [
    # lengths, H, Hkv, D, causal, out
    ([1], 1, 1, 64, True, "bf16"),
    ([64], 2, 2, 64, True, "bf16"),
    ([5, 0, 1, 128, 127, 129], 4, 2, 128, True, "bf16"),
    ([300, 17], 7, 1, 128, True, "fp16"),
    ([255, 256, 257], 8, 8, 64, False, "bf16"),
    ([0, 0, 3], 3, 3, 128, False, "int8"),
    ([512, 40, 700], 12, 4, 64, True, "int8"),
    ([1100], 16, 1, 128, True, "bf16"),
    ([513], 6, 3, 128, False, "fp16"),
    ([33] * 9, 5, 5, 64, True, "fp16"),
    ([641, 1281], 2, 1, 64, True, "bf16"),
    ([200], 32, 1, 128, True, "bf16"),
    ([90, 35], 130, 1, 64, True, "bf16"),
]


@pytest.mark.parametrize("lens,H,Hkv,D,causal,out", PACKED)
def test_packed_prompts(pkg, torch, lens, H, Hkv, D, causal, out):
    run_packed(pkg, torch, lens, None, H, Hkv, D, causal, out, seed=len(lens) + H + D)


@pytest.mark.parametrize("lens_q,lens_k,H,Hkv,D,causal,out", [
    ([3, 200, 1], [500, 100, 1], 4, 4, 64, True, "bf16"),        # fewer keys than tokens: the first tokens see none
    ([3, 0, 77], [0, 50, 333], 6, 2, 128, False, "bf16"),        # no keys at all, no tokens at all
    ([130, 300], [129, 40], 8, 1, 128, True, "int8"),
    ([1, 1, 1, 1], [1, 2, 1000, 129], 8, 2, 128, True, "fp16"),
    ([256], [2048], 4, 1, 64, True, "fp16"),
])
def test_packed_with_other_keys_than_queries(pkg, torch, lens_q, lens_k, H, Hkv, D, causal, out):
    run_packed(pkg, torch, lens_q, lens_k, H, Hkv, D, causal, out, seed=5)


def test_packed_views_of_a_fused_projection_and_generous_bounds(pkg, torch):
    run_packed(pkg, torch, [100, 260, 9], None, 6, 2, 128, True, "bf16", seed=3, fused=True, max_q=4096, max_k=100000)
    run_packed(pkg, torch, [100, 260, 9], None, 6, 2, 64, True, "bf16", seed=3, fused=True, max_k=0)


def test_more_sequences_than_a_warp_has_lanes(pkg, torch):
    lens = [(37 * i) % 150 for i in range(75)]
    run_packed(pkg, torch, lens, None, 4, 2, 64, True, "bf16", seed=1)
    run_packed(pkg, torch, [300] * 33, None, 8, 2, 128, True, "bf16", seed=2)
    run_paged(pkg, torch, [1 + i % 40 for i in range(70)], [60 + 3 * i for i in range(70)], 6, 2, 64, 16, "bf16", seed=3)
    run_paged(pkg, torch, [1] * 150, [1 + (61 * i) % 500 for i in range(150)], 8, 2, 128, 16, "fp16", seed=4)


@pytest.mark.parametrize("H,Hkv,D,causal", [(8, 1, 64, True), (4, 2, 128, False)])
def test_hundreds_of_sequences_some_of_them_empty(pkg, torch, H, Hkv, D, causal):
    """Units are found among the sequences in lots of 32: lots without a unit, one long sequence among short ones, ends inside a lot."""
    lens = [0] * 70 + [(53 * i) % 90 for i in range(150)] + [700] + [0] * 40 + [1, 33, 200] + [20] * 60 + [0] * 33 + [129]
    run_packed(pkg, torch, lens, None, H, Hkv, D, causal, "bf16", seed=D)


def run_mixed(pkg, torch, lens_q, lens_k, max_q, H, Hkv, D, out, seed, causal=True):
    """As run_paged, with a bound of the tokens that need not be reached; how many launches it took."""
    kc, vc, table, lens = make_cache(torch, lens_k, Hkv, D, 32, seed)
    T = sum(lens_q) + 2
    q = codes((T, H, D), seed + 5)
    o = torch.full((T, H, D), FILL[out], dtype=TYPES[out], device="cuda")
    before = pkg.launch_count()
    pkg.FMHAInferI8Paged(None, param(pkg), pkg.AttnDataDescriptorGrouped(len(lens_q), max_q, max(lens_k), H, Hkv, D), q, kc, vc, table, lens, starts(lens_q), o, causal=causal)
    launches = pkg.launch_count() - before
    at = 0
    for b, (n, m) in enumerate(zip(lens_q, lens_k)):
        want, spread = attention64(q[at:at + n], keys_of(kc, table, b, m), keys_of(vc, table, b, m), AMAX, causal)
        check(o[at:at + n], want, spread, m, out, AMAX, O_AMAX, max_q * H // Hkv, f"sequence {b}: {n} tokens on {m} keys", own=n * H // Hkv)
        at += n
    assert bool((o[at:] == FILL[out]).all())
    return launches


# (the launches that a B200 with 148 SMs makes: one, or the single tokens' and the chunks', or a third for more units than were expected)
MIXED = [
    # tokens of the sequences that bring many, (bound), sequences with few, most keys, H, Hkv, D, out
    ([480], 480, 32, 3000, 16, 2, 64, "bf16"),
    ([300, 17, 120], 300, 61, 2100, 32, 8, 128, "bf16"),
    ([300, 200], 300, 70, 1500, 8, 2, 128, "int8"),
    ([200] * 3, 1000, 30, 8000, 24, 2, 64, "fp16"),
    ([3] * 60, 700, 2, 3000, 32, 8, 128, "bf16"),          # not one that brings many: three tokens each are twelve rows
    ([40] * 90, 900, 0, 2500, 16, 4, 64, "bf16"),          # a bound that nobody reaches: many more units than were expected
    ([], 2000, 64, 4000, 32, 8, 128, "fp16"),              # nothing but single tokens
]


@pytest.mark.parametrize("many,max_q,few,keys,H,Hkv,D,out", MIXED)
def test_paged_single_tokens_among_chunks(pkg, torch, many, max_q, few, keys, H, Hkv, D, out):
    most = max(1, (8 if H // Hkv <= 8 else 16) * Hkv // H)              # tokens that the kernel for few rows takes
    lens_q = [1 + i % most if i % 11 else 0 for i in range(few)]
    for i, n in enumerate(many):
        lens_q.insert((7 * i) % (len(lens_q) + 1), n)
    lens_k = [keys if b == len(lens_q) // 2 else n + (277 * b) % (keys - n) for b, n in enumerate(lens_q)]
    assert run_mixed(pkg, torch, lens_q, lens_k, max_q, H, Hkv, D, out, seed=H + keys) > 1


@pytest.mark.parametrize("causal", [True, False])
def test_paged_a_token_more_than_the_kernel_for_few_rows_takes(pkg, torch, causal):
    for G, tokens in ((2, (4, 5)), (3, (2, 3)), (8, (1, 2)), (16, (1, 2)), (1, (8, 9))):
        lens_q = [tokens[i % 2] for i in range(60)] + [400]
        run_mixed(pkg, torch, lens_q, [900 + 31 * i for i in range(61)], 400, 4 * G, 4, 64, "bf16", seed=G, causal=causal)


def test_a_chunk_longer_than_its_bound_in_a_mixed_batch(pkg, torch):
    """It is computed in full, as in a batch of chunks alone, and nothing is reported (the fixture looks)."""
    assert run_mixed(pkg, torch, [1] * 20 + [480] + [1] * 20, [2000 + 50 * b for b in range(41)], 400, 16, 2, 64, "bf16", seed=12) > 1


# On 148 SMs 65 sequences stay in one launch -- 22 steps apart, 8 of them the launches, against 22 -- while 193 do not: 12 + 8 + 66 against 168.
@pytest.mark.parametrize("lots,apart", [(16, False), (48, True)])
def test_packed_single_tokens_among_chunks(pkg, torch, lots, apart):
    lens_q, lens_k, H, Hkv, D = [1, 2, 0, 1] * lots + [350], [40 + 17 * i for i in range(4 * lots)] + [1100], 16, 4, 128
    q, k, v = codes((sum(lens_q), H, D), 1), codes((sum(lens_k), Hkv, D), 2), codes((sum(lens_k), Hkv, D), 3)
    o = torch.full((sum(lens_q), H, D), 77.0, dtype=torch.bfloat16, device="cuda")
    before = pkg.launch_count()
    pkg.FMHAInferI8Packed(None, param(pkg), pkg.AttnDataDescriptorGrouped(4 * lots + 1, 350, max(lens_k), H, Hkv, D), q, k, v, starts(lens_q), starts(lens_k), o)
    assert (pkg.launch_count() - before > 1) == apart
    i = j = 0
    for n, m in zip(lens_q, lens_k):
        want, spread = attention64(q[i:i + n], k[j:j + m], v[j:j + m], AMAX, True)
        check(o[i:i + n], want, spread, m, "bf16", AMAX, O_AMAX, 350 * H // Hkv, f"{n} tokens on {m} keys", own=n * H // Hkv)
        i, j = i + n, j + m


def test_a_captured_mixed_step_follows_its_lengths(pkg, torch):
    """The same call with other lengths on the device: chunks where single tokens were, and the other way round."""
    B, H, Hkv, D, T, max_q = 40, 16, 4, 128, 700, 400
    lens_k = [2500 - 13 * b for b in range(B)]
    kc, vc, table, lens = make_cache(torch, lens_k, Hkv, D, 64, 3)
    q = codes((T, H, D), 8)
    o = torch.zeros((T, H, D), dtype=torch.bfloat16, device="cuda")
    cu = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
    args = (param(pkg), pkg.AttnDataDescriptorGrouped(B, max_q, 2500, H, Hkv, D), q, kc, vc, table, lens, cu, o)
    pkg.FMHAInferI8Paged(None, *args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.FMHAInferI8Paged(torch.cuda.current_stream().cuda_stream, *args)
    for lens_q in ([1] * 39 + [400], [400] + [2] * 10 + [1] * 29, [17] * 40, [0] * 20 + [1] * 20, [200, 3, 200] + [1] * 37):
        cu.copy_(starts(lens_q))
        o.fill_(77.0)
        graph.replay()
        at = 0
        for b, n in enumerate(lens_q):
            want, spread = attention64(q[at:at + n], keys_of(kc, table, b, lens_k[b]), keys_of(vc, table, b, lens_k[b]), AMAX, True)
            check(o[at:at + n], want, spread, lens_k[b], "bf16", AMAX, O_AMAX, max_q * H // Hkv, f"{n} tokens", own=n * H // Hkv)
            at += n
        assert bool((o[at:] == 77.0).all())


def test_more_keys_than_waits_are_sized_for(pkg, torch):
    """Chunks on more than 2^26 keys are refused, single tokens are not; a bound that the tensors do not reach does not count."""
    kc = torch.zeros((1, 1, 4096, 64), dtype=torch.int8, device="cuda")
    q = torch.zeros((40, 1, 64), dtype=torch.int8, device="cuda")
    o = torch.empty((40, 1, 64), dtype=torch.bfloat16, device="cuda")
    lens = torch.tensor([50], dtype=torch.int32, device="cuda")
    for width, tokens, most, refused in ((1 << 15, 40, 1 << 27, True), (1 << 15, 40, (1 << 26) + 1, True), (1 << 15, 40, 1 << 26, False), (1 << 15, 4, 1 << 27, False),
                                         (1 << 14, 40, 1 << 27, False)):
        table = torch.zeros((1, width), dtype=torch.int32, device="cuda")
        args = (None, param(pkg), pkg.AttnDataDescriptorGrouped(1, tokens, most, 1, 1, 64), q[:tokens], kc, kc, table, lens, starts([tokens]), o[:tokens])
        if refused:
            with pytest.raises(pkg.FmhaError) as e:
                pkg.FMHAInferI8Paged(*args)
            assert e.value.status == pkg.ERR_TOO_LARGE
        else:
            o.fill_(7.0)
            pkg.FMHAInferI8Paged(*args)
            assert bool((o[:tokens] == 0).all())
    k = torch.zeros((50, 1, 64), dtype=torch.int8, device="cuda")
    o.fill_(7.0)
    pkg.FMHAInferI8Packed(None, param(pkg), pkg.AttnDataDescriptorGrouped(1, 40, 1 << 30, 1, 1, 64), q, k, k, starts([40]), starts([50]), o)
    assert bool((o == 0).all())


@pytest.mark.parametrize("out", ["bf16", "int8"])
def test_outputs_with_strides_and_the_least_alignment(pkg, torch, out):
    """o as a view with a row of its own spacing, 16-byte aligned only: the narrow stores, and nothing besides the rows is touched."""
    T, H, Hkv, D = 150, 6, 2, 64
    size = TYPES[out].itemsize
    q, k, v = codes((T, H, D), 1), codes((T, Hkv, D), 2), codes((T, Hkv, D), 3)
    flat = torch.full(((T + 1) * (H * D + 16 // size) + 64,), FILL[out], dtype=TYPES[out], device="cuda")
    o = flat[16 // size:].as_strided((T, H, D), (H * D + 16 // size, D, 1))
    assert o.data_ptr() % 32 == 16
    cu = starts([T])
    for tokens in (T, 1):
        before = flat.clone()
        desc = pkg.AttnDataDescriptorGrouped(1, tokens, T, H, Hkv, D)
        pkg.FMHAInferI8Packed(None, param(pkg), desc, q[:tokens], k, v, starts([tokens]), cu, o[:tokens])
        want, scales = attention64(q[:tokens], k, v, AMAX, True)
        check(o[:tokens], want, scales, T, out, AMAX, O_AMAX, tokens * 3)
        o[:tokens] = FILL[out] if tokens == T else before.as_strided((T, H, D), o.stride(), o.storage_offset())[:tokens]
        assert torch.equal(flat, before)


def test_no_tokens_and_no_keys(pkg, torch):
    """Calls in which nothing, or nothing but zeros, is to be written."""
    for D, H in ((64, 4), (128, 48)):                        # few rows, and more than sixteen
        desc = pkg.AttnDataDescriptorGrouped(2, 5, 5, H, 2, D)
        empty_k = codes((0, 2, D), 1)
        o = torch.full((5, H, D), 7.0, dtype=torch.bfloat16, device="cuda")
        pkg.FMHAInferI8Packed(None, param(pkg), desc, codes((5, H, D), 1), empty_k, empty_k, starts([2, 3]), starts([0, 0]), o)
        assert not bool(o.any())
        pkg.FMHAInferI8Packed(None, param(pkg), desc, codes((0, H, D), 1), empty_k, empty_k, starts([0, 0]), starts([0, 0]), o[:0])
        o.fill_(7.0)
        kc = codes((1, 2, 16, D), 2)
        lens = torch.zeros(2, dtype=torch.int32, device="cuda")
        pkg.FMHAInferI8Paged(None, param(pkg), desc, codes((5, H, D), 1), kc, kc, torch.zeros((2, 1), dtype=torch.int32, device="cuda"), lens, starts([1, 0]), o)
        assert not bool(o[0].any()) and bool((o[1:] == 7.0).all())


def test_packed_rows_that_are_far_from_even(pkg, torch):
    """Ranges so wide that a row's largest score takes everything, and so narrow that all keys count the same."""
    for a in (1e-9, 40.0, 250.0, 777.7, 1500.0, 1e9):
        amax = (a, a, AMAX[2])
        q, k, v = codes((150, 4, 64), 1), codes((150, 2, 64), 2), codes((150, 2, 64), 3)
        o = torch.empty((150, 4, 64), dtype=torch.bfloat16, device="cuda")
        cu = starts([150])
        pkg.FMHAInferI8Packed(None, pkg.FMHAParamI8(*amax, 1.0, 1.0), pkg.AttnDataDescriptorGrouped(1, 150, 150, 4, 2, 64), q, k, v, cu, cu, o)
        want, spread = attention64(q, k, v, amax, True)
        check(o, want, spread, 150, "bf16", amax, 1.0, 300, str(a))
        for tokens in (1, 8):                                # eight rows, and sixteen
            one = starts([tokens])
            pkg.FMHAInferI8Packed(None, pkg.FMHAParamI8(*amax, 1.0, 1.0), pkg.AttnDataDescriptorGrouped(1, tokens, 150, 4, 2, 64), q[:tokens], k, v, one, cu, o[:tokens])
            want, spread = attention64(q[:tokens], k, v, amax, True)
            check(o[:tokens], want, spread, 150, "bf16", amax, 1.0, 2 * tokens, f"{a}, {tokens}")


def test_packed_identical_scores_and_growing_maxima(pkg, torch):
    """Keys in ascending order of their scores: the running maximum grows with every tile, by little and by much."""
    D, n = 64, 900
    for step in (0.02, 1.0):
        q = torch.full((1, 1, D), 100, dtype=torch.int8, device="cuda")
        k = torch.zeros((n, 1, D), dtype=torch.int8, device="cuda")
        level = (torch.arange(n, device="cuda") * step).long()
        for i in range(D):
            k[:, 0, i] = (level // D + (level % D > i)).clamp(-127, 127).to(torch.int8)
        v = codes((n, 1, D), 9)
        o = torch.empty((1, 1, D), dtype=torch.float16, device="cuda")
        pkg.FMHAInferI8Packed(None, param(pkg), pkg.AttnDataDescriptorGrouped(1, 1, n, 1, 1, D), q, k, v, starts([1]), starts([n]), o)
        want, spread = attention64(q, k, v, AMAX, True)
        check(o, want, spread, n, "fp16", AMAX, 1.0, 1, str(step))
        rows = q.expand(400, 1, D).contiguous()
        o = torch.empty((400, 1, D), dtype=torch.float16, device="cuda")
        pkg.FMHAInferI8Packed(None, param(pkg), pkg.AttnDataDescriptorGrouped(1, 400, n, 1, 1, D), rows, k, v, starts([400]), starts([n]), o)
        want, spread = attention64(rows, k, v, AMAX, True)
        check(o, want, spread, n, "fp16", AMAX, 1.0, 400, str(step))


def test_packed_offsets_outside_the_tensors_are_cut_and_reported(pkg, torch):
    q, k, v = codes((20, 2, 64), 1), codes((20, 2, 64), 2), codes((20, 2, 64), 3)
    desc = pkg.AttnDataDescriptorGrouped(2, 16, 16, 2, 2, 64)
    for cu in ([0, 10, 25], [-3, 10, 20], [0, 12, 8]):
        o = torch.zeros((21, 2, 64), dtype=torch.bfloat16, device="cuda")
        t = torch.tensor(cu, dtype=torch.int32, device="cuda")
        pkg.FMHAInferI8Packed(None, param(pkg), desc, q, k, v, t, t, o[:20])
        st, words = pkg.device_status()
        assert st == pkg.ERR_DEVICE and words[0] == 13 and words[2] == 0, cu
        assert not bool(o[20].any())
    # more tokens than max_seq_q says: reported
    cu = starts([20, 0])
    o = torch.zeros((20, 2, 64), dtype=torch.bfloat16, device="cuda")
    pkg.FMHAInferI8Packed(None, param(pkg), pkg.AttnDataDescriptorGrouped(2, 4, 20, 2, 2, 64), q, k, v, cu, cu, o)
    st, words = pkg.device_status()
    assert st == pkg.ERR_DEVICE and words[0] == 13


# ------------------------------------------------------------------------------------------------ paged cache

def make_cache(torch, lens, Hkv, D, page, seed, together=False, wide=0):
    wanted = [-(-n // page) for n in lens]
    pages = sum(wanted) + 2
    if together:
        both = codes((pages, 2, Hkv, page, D), seed)
        kc, vc = both[:, 0], both[:, 1]
    else:
        kc, vc = codes((pages, Hkv, page, D), seed), codes((pages, Hkv, page, D), seed + 1)
    g = torch.Generator()
    g.manual_seed(seed)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table, at = torch.full((len(lens), max(wanted + [1]) + wide), -7, dtype=torch.int32), 0      # entries that nobody may read
    for b, n in enumerate(wanted):
        table[b, :n] = order[at:at + n]
        at += n
    return kc, vc, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


def keys_of(cache, table, b, n):
    page = cache.shape[2]
    rows = table[b, :-(-n // page)].long()
    return cache[rows].transpose(1, 2).reshape(-1, cache.shape[1], cache.shape[3])[:n]


def run_paged(pkg, torch, lens_q, lens_k, H, Hkv, D, page, out, seed, causal=True, tail=2, together=False, max_k=None, wide=0):
    kc, vc, table, lens = make_cache(torch, lens_k, Hkv, D, page, seed, together, wide)
    T = sum(lens_q) + tail
    q = codes((T, H, D), seed + 5)
    o = torch.full((T, H, D), FILL[out], dtype=TYPES[out], device="cuda")
    desc = pkg.AttnDataDescriptorGrouped(len(lens_q), max(lens_q), max(lens_k) if max_k is None else max_k, H, Hkv, D)
    pkg.FMHAInferI8Paged(None, param(pkg), desc, q, kc, vc, table, lens, starts(lens_q), o, causal=causal)
    at = 0
    for b, (n, m) in enumerate(zip(lens_q, lens_k)):
        want, spread = attention64(q[at:at + n], keys_of(kc, table, b, m), keys_of(vc, table, b, m), AMAX, causal)
        check(o[at:at + n], want, spread, m, out, AMAX, O_AMAX, desc.max_seq_q * H // Hkv, f"sequence {b}: {n} tokens on {m} keys", own=n * H // Hkv)
        at += n
    assert bool((o[at:] == FILL[out]).all())


PAGED = [
    # tokens, keys, H, Hkv, D, page, out
    ([1], [1], 1, 1, 64, 16, "bf16"),
    ([1], [1025], 32, 8, 128, 16, "bf16"),
    ([1, 1, 1, 1, 1], [1, 16, 17, 0, 1000], 8, 2, 128, 16, "bf16"),
    ([1] * 6, [127, 128, 129, 255, 256, 257], 7, 1, 64, 32, "fp16"),
    ([1, 1], [5000, 3], 28, 4, 128, 64, "int8"),
    ([1, 1, 1], [4097, 12000, 100], 4, 4, 64, 128, "bf16"),
    ([1], [20011], 16, 1, 128, 16, "fp16"),
    ([2, 1, 4], [200, 1, 900], 4, 2, 128, 256, "bf16"),
    ([1, 100, 1, 0, 37], [700, 900, 64, 10, 37], 8, 2, 64, 16, "bf16"),
    ([300], [300], 4, 1, 128, 32, "int8"),
    ([129, 1], [2000, 2000], 12, 3, 128, 64, "fp16"),
    ([64], [16384], 8, 1, 128, 16, "bf16"),
    ([5], [3], 6, 2, 64, 16, "bf16"),
    ([520, 1, 1], [1300, 7, 513], 16, 2, 64, 4096, "bf16"),
    ([1, 1], [9000, 8999], 40, 1, 64, 16, "bf16"),
    ([3, 1], [700, 2000], 10, 2, 128, 16, "fp16"),
    ([7], [30001], 24, 3, 64, 32, "bf16"),
    ([40, 2], [9001, 5], 8, 4, 128, 16, "fp16"),
    ([100], [70000], 2, 1, 128, 64, "bf16"),
]


@pytest.mark.parametrize("lens_q,lens_k,H,Hkv,D,page,out", PAGED)
def test_paged(pkg, torch, lens_q, lens_k, H, Hkv, D, page, out):
    run_paged(pkg, torch, lens_q, lens_k, H, Hkv, D, page, out, seed=H + D + page)


# Up to 32 rows to a key head, on either side of what the kernels' choice looks at: rows (16, 17, 32, 33), key tiles (7, 8) and, for head_dim 128, the number of units.
FEW_ROWS = [
    # sequences, most tokens, most keys, H, Hkv, D, out
    (3, 17, 300, 4, 4, 64, "bf16"),
    (3, 8, 1500, 8, 2, 64, "fp16"),
    (2, 11, 700, 6, 2, 64, "int8"),
    (5, 1, 2100, 34, 2, 64, "bf16"),
    (70, 8, 900, 32, 8, 128, "bf16"),
    (70, 8, 897, 32, 8, 128, "int8"),
    (70, 8, 896, 32, 8, 128, "bf16"),
    (62, 17, 1100, 8, 8, 128, "fp16"),
    (70, 11, 900, 24, 8, 128, "bf16"),
    (40, 1, 1000, 320, 16, 128, "fp16"),
]


@pytest.mark.parametrize("sequences,tokens,keys,H,Hkv,D,out", FEW_ROWS)
def test_paged_up_to_32_rows(pkg, torch, sequences, tokens, keys, H, Hkv, D, out):
    lens_q = [tokens if b % 3 == 0 else (5 * b + 1) % (tokens + 1) for b in range(sequences)]
    lens_k = [keys if b == 0 else n + (131 * b) % (keys + 1 - n) for b, n in enumerate(lens_q)]
    run_paged(pkg, torch, lens_q, lens_k, H, Hkv, D, 32, out, seed=sequences + tokens)


@pytest.mark.parametrize("D,sequences,keys", [(64, 4, 40), (128, 64, 930)])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_up_to_32_rows(pkg, torch, D, sequences, keys, causal):
    lens_q = [(b * 7 + 8) % 9 for b in range(sequences)]
    run_packed(pkg, torch, lens_q, [keys if b == 1 else (b * 97) % keys for b in range(sequences)], 24, 8, D, causal, "bf16", seed=D, max_q=9)


def test_paged_other_forms(pkg, torch):
    run_paged(pkg, torch, [1, 50, 1], [333, 444, 5], 6, 3, 128, 16, "bf16", seed=1, together=True)
    run_paged(pkg, torch, [1, 50, 1], [333, 444, 5], 6, 3, 64, 32, "bf16", seed=2, causal=False)
    run_paged(pkg, torch, [1, 1, 1], [333, 444, 5], 6, 3, 64, 32, "bf16", seed=3, wide=500, max_k=16000)     # bounds far beyond the lengths
    run_paged(pkg, torch, [1, 1, 1], [3330, 4440, 5], 6, 3, 128, 32, "bf16", seed=4, max_k=1)                  # and far below


def test_paged_many_keys_for_one_warp(pkg, torch):
    """A bound far below the length leaves one CTA to go through all keys: the whole-number sums of a warp fill up more than once."""
    D, page, n = 128, 4096, 300000
    kc, vc = codes((3, 1, page, D), 1), codes((3, 1, page, D), 2)
    table = (torch.arange(-(-n // page), device="cuda") % 3).to(torch.int32)[None].contiguous()      # the same pages over and over
    q, o = codes((1, 4, D), 3), torch.empty((1, 4, D), dtype=torch.float16, device="cuda")
    pkg.FMHAInferI8Paged(None, param(pkg), pkg.AttnDataDescriptorGrouped(1, 1, 1, 4, 1, D), q, kc, vc, table, torch.tensor([n], dtype=torch.int32, device="cuda"), starts([1]), o)
    want, scales = attention64(q, keys_of(kc, table, 0, n), keys_of(vc, table, 0, n), AMAX, True)
    check(o, want, scales, n, "fp16", AMAX, 1.0, 4)


def test_paged_pages_and_lengths_outside_are_reported(pkg, torch):
    kc, vc, table, lens = make_cache(torch, [300, 40], 2, 64, 16, 1)
    q, o = codes((2, 2, 64), 2), torch.zeros((2, 2, 64), dtype=torch.bfloat16, device="cuda")
    desc = pkg.AttnDataDescriptorGrouped(2, 1, 300, 2, 2, 64)
    for bad in (kc.shape[0], -1, 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[0, 3] = bad
        pkg.FMHAInferI8Paged(None, param(pkg), desc, q, kc, vc, t, lens, starts([1, 1]), o)
        st, words = pkg.device_status()
        assert st == pkg.ERR_DEVICE and words[0] == 13 and words[2] == 1, (bad, words)
        want, spread = attention64(q[1:], keys_of(kc, table, 1, 40), keys_of(vc, table, 1, 40), AMAX, True)
        check(o[1:], want, spread, 40, "bf16", AMAX, O_AMAX, 1)
    for length in (table.shape[1] * 16 + 1, -1):
        pkg.FMHAInferI8Paged(None, param(pkg), desc, q, kc, vc, table.clamp(min=0), torch.tensor([length, 40], dtype=torch.int32, device="cuda"), starts([1, 1]), o)
        st, words = pkg.device_status()
        assert st == pkg.ERR_DEVICE and words[0] == 13 and words[2] == 0, words
        check(o[1:], want, spread, 40, "bf16", AMAX, O_AMAX, 1)


def test_paged_offsets_beyond_32_bits(pkg, torch):
    """A cache of more than 2^32 bytes: the last pages are found."""
    Hkv, page, D = 8, 256, 128
    pages = 2 ** 32 // (Hkv * page * D) + 40
    kc = torch.zeros((pages, Hkv, page, D), dtype=torch.int8, device="cuda")
    n = 600
    table = torch.tensor([[pages - 1, 5, pages - 17]], dtype=torch.int32, device="cuda")
    k, v, g = codes((n, Hkv, D), 1), codes((n, Hkv, D), 2), 2
    vc = torch.zeros_like(kc)
    for cache, x in ((kc, k), (vc, v)):
        for i in range(3):
            part = x[i * page:(i + 1) * page]
            cache[int(table[0, i]), :, :part.shape[0]] = part.transpose(0, 1)
    for n_q in (1, 200):
        q, o = codes((n_q, Hkv * g, D), 3), torch.empty((n_q, Hkv * g, D), dtype=torch.bfloat16, device="cuda")
        pkg.FMHAInferI8Paged(None, param(pkg), pkg.AttnDataDescriptorGrouped(1, n_q, n, Hkv * g, Hkv, D), q, kc, vc, table,
                             torch.tensor([n], dtype=torch.int32, device="cuda"), starts([n_q]), o)
        want, spread = attention64(q, k, v, AMAX, True)
        check(o, want, spread, n, "bf16", AMAX, O_AMAX, n_q * g)


# ------------------------------------------------------------------------------------------------ together, as they are used

def test_prefill_then_chunks_then_single_tokens_agree(pkg, torch):
    """One model layer: a whole prompt through the packed call, and the same tokens in chunks and one by one through the cache."""
    T, H, Hkv, D, page, rot = 300, 8, 2, 128, 16, 64
    qf, kf, vf = make_qkv(torch, T, H, Hkv, D, "bf16", 11)
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    freq, table = make_table(pkg, torch, rot, T)
    q8 = torch.empty((T, H, D), dtype=torch.int8, device="cuda")
    k8, v8 = (torch.empty((T, Hkv, D), dtype=torch.int8, device="cuda") for _ in range(2))
    pkg.rope_quantize_append(None, param(pkg), qf, kf, vf, pos, table, q8, k8, v8)
    whole = torch.empty((T, H, D), dtype=torch.bfloat16, device="cuda")
    cu = starts([T])
    pkg.FMHAInferI8Packed(None, param(pkg), pkg.AttnDataDescriptorGrouped(1, T, T, H, Hkv, D), q8, k8, v8, cu, cu, whole)
    want_q, want_k = (quantise64(rotate64(x.double(), pos, freq, 1.0, False), a) for x, a in ((qf, AMAX[0]), (kf, AMAX[1])))
    want, spread = attention64(want_q, want_k, quantise64(vf.double(), AMAX[2]), AMAX, True)
    check(whole, want, spread, T, "bf16", AMAX, 1.0, T * H // Hkv)

    pages = -(-T // page)
    kc, vc = (torch.zeros((pages + 1, Hkv, page, D), dtype=torch.int8, device="cuda") for _ in range(2))
    page_table = torch.randperm(pages + 1, device="cuda")[:pages].to(torch.int32)[None]
    out = torch.empty_like(whole)
    at, rows_of = 0, []
    for n in (129, 70, 33, 3) + (1,) * 65:
        rows = slice(at, at + n)
        where = torch.arange(at, at + n, device="cuda")
        slots = page_table[0, where // page].long() * page + where % page
        qn = torch.empty((n, H, D), dtype=torch.int8, device="cuda")
        pkg.rope_quantize_append(None, param(pkg), qf[rows], kf[rows], vf[rows], pos[rows], table, qn, kc, vc, slots=slots)
        rows_of.append((rows, n * H // Hkv))
        at += n
        pkg.FMHAInferI8Paged(None, param(pkg), pkg.AttnDataDescriptorGrouped(1, n, at, H, Hkv, D), qn, kc, vc, page_table,
                             torch.tensor([at], dtype=torch.int32, device="cuda"), starts([n]), out[rows])
    assert at == T
    for rows, n in rows_of:
        check(out[rows], want[rows], tuple(x[rows] for x in spread), T, "bf16", AMAX, 1.0, n)


def test_a_captured_step_follows_lengths_and_pages(pkg, torch):
    """Append and attention of a decoding step in one graph; between replays the lengths, slots, pages and inputs change in place."""
    B, H, Hkv, D, page = 3, 8, 2, 64, 16
    kc, vc, table, lens = make_cache(torch, [40, 700, 129], Hkv, D, page, 21, wide=3)
    table.clamp_(min=0)
    qkv = torch.randn((B, H + 2 * Hkv, D), device="cuda").bfloat16()
    freq, rotations = make_table(pkg, torch, D, 4096)
    pos, slots = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int64, device="cuda")
    q8 = torch.empty((B, H, D), dtype=torch.int8, device="cuda")
    o = torch.empty((B, H, D), dtype=torch.bfloat16, device="cuda")
    cu = starts([1] * B)
    desc = pkg.AttnDataDescriptorGrouped(B, 1, table.shape[1] * page, H, Hkv, D)

    def step():
        pkg.rope_quantize_append(None, param(pkg), qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:], pos, rotations, q8, kc, vc, slots=slots)
        pkg.FMHAInferI8Paged(None, param(pkg), desc, q8, kc, vc, table, lens, cu, o)

    def place(new):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        pos.copy_(lens - 1)
        slots.copy_(table[torch.arange(B, device="cuda"), (pos // page).long()].long() * page + pos % page)
        qkv.normal_()

    place([40, 700, 129])
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                       # two graphs of the same call live side by side
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append(g)
    for i, new in enumerate(([40, 700, 129], [41, 701, 1], [1, 640, 144], [48, 720, 130])):
        place(new)
        o.zero_()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        for b, n in enumerate(new):
            want, spread = attention64(q8[b:b + 1], keys_of(kc, table, b, n), keys_of(vc, table, b, n), AMAX, True)
            check(o[b:b + 1], want, spread, n, "bf16", AMAX, O_AMAX, H // Hkv, f"replay {i}")
            assert torch.equal(keys_of(vc, table, b, n)[-1], quantise64(qkv[b, H + Hkv:].double(), AMAX[2]))


def test_calls_on_two_streams_at_once_and_in_a_row(pkg, torch):
    """The same bytes as alone, for calls side by side on two streams and calls that start while the one before drains."""
    args = []
    for seed, (H, Hkv, D) in enumerate(((8, 2, 128), (12, 4, 64))):
        lens = [700, 3, 260]
        q, k, v, o = run_packed(pkg, torch, lens, None, H, Hkv, D, True, "bf16", seed=seed)
        args.append((pkg.AttnDataDescriptorGrouped(3, 700, 700, H, Hkv, D), q, k, v, starts(lens), o))
    streams = [torch.cuda.Stream() for _ in args]
    outs = [[torch.zeros_like(a[5]) for _ in range(20)] for a in args]
    torch.cuda.synchronize()
    for i in range(20):
        for s, (desc, q, k, v, cu, o), out in zip(streams, args, outs):
            pkg.FMHAInferI8Packed(s, param(pkg), desc, q, k, v, cu, cu, out[i])
    torch.cuda.synchronize()
    for (desc, q, k, v, cu, o), out in zip(args, outs):
        n = 700 + 3 + 260
        for x in out:
            assert torch.equal(x[:n], o[:n])


def test_host_threads_call_at_once(pkg, torch):
    """Four host threads, each with a stream, shapes and a cache of its own."""
    import threading
    failures = []

    def work(i):
        try:
            torch.cuda.set_device(0)
            with torch.cuda.stream(torch.cuda.Stream()):
                for rep in range(5):
                    run_paged(pkg, torch, [1, 20 * i, 3], [100 + i, 400, 3], 4 * (i + 1), 2, (64, 128)[i % 2], 16, "bf16", seed=10 * i + rep)
                    run_packed(pkg, torch, [50 * i + 1, 7], None, 4, 2, (128, 64)[i % 2], True, "bf16", seed=rep)
        except BaseException as e:  # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures[0]


def test_plain_calls_give_the_same_bytes_every_time(pkg, torch):
    q, k, v, o = run_packed(pkg, torch, [700, 300], None, 8, 2, 128, True, "bf16", seed=4)
    kc, vc, table, lens = make_cache(torch, [5000, 900], 2, 128, 16, 4)
    table.clamp_(min=0)
    cu = starts([700, 300])
    first = None
    for _ in range(5):
        again = torch.empty_like(o)
        pkg.FMHAInferI8Packed(None, param(pkg), pkg.AttnDataDescriptorGrouped(2, 700, 700, 8, 2, 128), q, k, v, cu, cu, again)
        assert torch.equal(again[:1000], o[:1000])
        one = torch.empty((2, 8, 128), dtype=torch.bfloat16, device="cuda")
        pkg.FMHAInferI8Paged(None, param(pkg), pkg.AttnDataDescriptorGrouped(2, 1, 5000, 8, 2, 128), q[:2], kc, vc, table, lens, starts([1, 1]), one)
        first = one if first is None else first
        assert torch.equal(one, first)
