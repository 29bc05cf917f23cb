"""GPU tests of the serving attention where one key takes most of a row's weight and many others share the rest, as a first token does in trained causal
models.  What the others add to the output must survive the rounding of P, whichever kernel has the row."""
import math

import pytest

from _serving import AMAX, TYPES, starts

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(600)]
TILE = 128


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


def scale_of(D):
    return AMAX[0] * AMAX[1] / 127.0 ** 2 / math.sqrt(D)


def peaked(torch, tokens, keys, H, Hkv, D, nats, sinks, spread, value, seed):
    """q, k, v in codes: key `sinks[i]` lies `nats` above the others in every row, whose logits are normal with deviation `spread`.  32 columns make the
    difference -- 127 in every q, t in those keys -- and the others the rest.  value: what the others' v is around, sinks have v = 0; or a constant for all keys."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c = scale_of(D)
    std = math.sqrt(spread / (c * math.sqrt(D - 32)))                # of q and k, for scores of that deviation
    q = (torch.randn((tokens, H, D), device="cuda", generator=g) * std).round().clamp(-127, 127).to(torch.int8)
    k = (torch.randn((keys, Hkv, D), device="cuda", generator=g) * std).round().clamp(-127, 127).to(torch.int8)
    q[..., :32], k[..., :32] = 127, 0
    level = nats / (c * 127.0)                                       # the sum of those columns
    columns = torch.tensor([int(level // 32) + (i < level % 32) for i in range(32)], device="cuda").clamp(max=127).to(torch.int8)
    if value is None:
        v = torch.full((keys, Hkv, D), 100, dtype=torch.int8, device="cuda")
    else:
        v = torch.randint(value - 20, value + 21, (keys, Hkv, D), dtype=torch.int8, device="cuda", generator=g)
    for s in sinks:
        k[s, :, 32:] = 0
        k[s, :, :32] = columns
        if value is not None:
            v[s] = 0
    return q, k, v


def bounded(torch, o, q, k, v, o_type, n_chain, what):
    """One sequence, causal.  In real units |o - exact| <=
      output   half a step of its type, relative
      P        fp16 (more than eight rows): half a step, 2^-11 of p |v|; what it is relative to is 2^7 of fp16's units or more, so that the smallest half a step,
               2^-25, is 2^-32 of that, which is the row's largest p at most.
               Up to eight rows, for each tile of 128 keys in which the row sees n: half a step of 16 bits, 2^-17 of the tile's largest p, for each of its keys where
               their p, none counted with more than 2^-5 of that, add up to n 2^-7 and more: 2^-10 of that sum times the mean |v|.  Half a step of 32 bits otherwise.
      exp2     2^-18 of every p, once above and once below the line of the quotient (as in _serving.tolerance)
      sums     2^-24 for every addition that a term goes through, above and below."""
    n, H, D = q.shape
    m, Hkv = k.shape[0], k.shape[1]
    G = H // Hkv
    c = float(torch.tensor(AMAX[0])) * float(torch.tensor(AMAX[1])) / 127.0 ** 2 / math.sqrt(D)
    real = float(torch.tensor(AMAX[2])) / 127.0
    for h in range(Hkv):
        kk, vv = k[:, h].double(), v[:, h].double()
        s = (q[:, h * G:(h + 1) * G].reshape(-1, D).double() @ kk.T) * c
        seen = torch.ones((n, m), dtype=torch.bool, device="cuda").tril(m - n).repeat_interleave(G, 0)
        s = s.masked_fill(~seen, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        l = p.sum(-1, keepdim=True)
        want, each = p @ vv / l * real, p @ vv.abs() / l * real
        if n * G > 8:
            of_p = each * 2.0 ** -11 + seen.double() @ vv.abs() / l * (2.0 ** -32 * real)
        else:
            tiles = torch.nn.functional.pad(p, (0, -m % TILE)).view(n * G, -1, TILE)
            top = tiles.amax(-1, keepdim=True)
            bound = torch.minimum(tiles, top * 2.0 ** -5).sum(-1) * 2.0 ** -10 + top[..., 0] * 2.0 ** -26
            keys = torch.nn.functional.pad(seen.double(), (0, -m % TILE)).view(n * G, -1, TILE)
            mean = torch.einsum("rtk,tkd->rtd", keys, torch.nn.functional.pad(vv.abs(), (0, 0, 0, -m % TILE)).view(-1, TILE, D)) / keys.sum(-1, keepdim=True).clamp(min=1)
            of_p = (bound[..., None] * mean).sum(1) / l * real
        got = o[:, h * G:(h + 1) * G].reshape(-1, D).double()
        tol = want.abs() * (torch.finfo(TYPES[o_type]).eps / 2) * 1.001 + of_p * 1.005 + each * (2.0 ** -17 + n_chain * 2.0 ** -23) + 2.0 ** -25
        worst = float(((got - want).abs() / tol).max())
        assert worst <= 1.0, f"{what}, key head {h}: {worst:.3g} times the tolerance; mean of the output {float(got.mean()):.5g}, exact {float(want.mean()):.5g}"


def paged(pkg, torch, q, k, v, o_type, max_k, page=64):
    n, H, D = q.shape
    m, Hkv = k.shape[0], k.shape[1]
    pages = -(-m // page)
    kc, vc = (torch.nn.functional.pad(x, (0, 0, 0, 0, 0, pages * page - m)).view(pages, page, Hkv, D).transpose(1, 2).contiguous() for x in (k, v))
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    o = torch.empty((n, H, D), dtype=TYPES[o_type], device="cuda")
    pkg.FMHAInferI8Paged(None, pkg.FMHAParamI8(*AMAX, 1.0, 1.0), pkg.AttnDataDescriptorGrouped(1, n, max_k, H, Hkv, D), q, kc, vc, table,
                         torch.tensor([m], dtype=torch.int32, device="cuda"), starts([n]), o)
    return o


# A bound of one key keeps a unit on one CTA (two warps at head_dim 128, four at 64), the true one spreads it over a cluster of up to 8 or 16 CTAs (up to 48 warps and more).
@pytest.mark.parametrize("D,G", [(128, 4), (64, 8), (128, 1), (64, 3)])
@pytest.mark.parametrize("keys,nats,spread", [(8192, 12.5, 1.0), (32768, 12.5, 1.0), (131072, 12.5, 1.0), (131072, 13.0, 0.3), (20011, 8.0, 1.0), (32768, 16.0, 1.0), (32768, 22.0, 0.3),
                                              (20011, 12.0, 2.5)])
@pytest.mark.parametrize("alone", [True, False])
def test_single_tokens_keep_what_a_dominant_key_leaves(pkg, torch, D, G, keys, nats, spread, alone):
    for sinks, value in (([0], 20), ([0], None), ([0, 1, 2, 3], 20), ([0, keys // 2 + 5, keys - 1], -60)):
        q, k, v = peaked(torch, 1, keys, 2 * G, 2, D, nats, sinks, spread, value, seed=keys + D)
        o = paged(pkg, torch, q, k, v, "fp16", 1 if alone else keys)
        # (a warp adds a tile's output and sum in two parts at most, 16 terms of a lane, and 64 partial rows at the end)
        bounded(torch, o, q, k, v, "fp16", 2 * keys / TILE + 100, f"sinks {sinks}, values around {value}")


@pytest.mark.parametrize("D", [64, 128])
def test_single_tokens_with_a_dominant_key_in_every_tile(pkg, torch, D):
    """Every tile of 128 keys has a key that takes most of its weight, at any of its places, and heads differ in which."""
    keys, G = 3000, 7
    q, k, v = peaked(torch, 1, keys, G, 1, D, 0.0, [], 0.5, 50, seed=1)
    for i in range(keys // TILE + 1):
        at = min(i * TILE + (37 * i) % TILE, keys - 1)
        k[at] = 0
        k[at, 0, :32] = 3 + (7 * i) % 20
        v[at] = 0
    for most in (1, keys):
        bounded(torch, paged(pkg, torch, q, k, v, "fp16", most), q, k, v, "fp16", 2 * keys / TILE + 100, "a dominant key in every tile")
    # tokens of one sequence that see different parts of the last tiles, two to eight rows
    for n, H in ((2, 1), (3, 2), (4, 2), (8, 1)):
        q, k, v = peaked(torch, n, 1000, H, 1, D, 12.5, [0, 997], 1.0, 30, seed=n)
        bounded(torch, paged(pkg, torch, q, k, v, "fp16", 1000), q, k, v, "fp16", 200, f"{n} tokens")


@pytest.mark.parametrize("D", [64, 128])
def test_the_same_row_in_any_company(pkg, torch, D):
    """A token's output is the same within its roundings alone, among others and in a call of chunks."""
    keys, H, Hkv = 9000, 8, 2
    q, k, v = peaked(torch, 40, keys, H, Hkv, D, 12.5, [0], 1.0, 20, seed=D)
    last = slice(39, 40)
    alone = paged(pkg, torch, q[last], k, v, "fp16", keys)
    bounded(torch, alone, q[last], k, v, "fp16", 300, "alone")
    for n in (2, 4, 8, 40):                                  # eight rows, sixteen, 32, and the chunk kernel
        o = paged(pkg, torch, q[40 - n:], k, v, "fp16", keys)
        bounded(torch, o, q[40 - n:], k, v, "fp16", keys / 4, f"one of {n}")
        assert float((o[-1].double() - alone[0].double()).abs().max()) <= 2 * 2.0 ** -9 * float(alone.abs().max()), n


# Sixteen rows, 32 in two groups, and the chunk kernel: whole units, and units shared by clusters.
@pytest.mark.parametrize("D,H,Hkv,tokens", [(128, 4, 1, 4), (64, 16, 2, 1), (64, 8, 2, 8), (128, 12, 4, 40), (64, 6, 2, 70), (128, 8, 8, 300)])
@pytest.mark.parametrize("keys,nats", [(8192, 12.5), (30000, 16.0), (30000, 18.5)])
def test_more_rows_keep_what_a_dominant_key_leaves(pkg, torch, D, H, Hkv, tokens, keys, nats):
    for sinks, value in (([0], 20), ([0, 1, 2, 3], 50), ([0, keys // 2 + 5], None)):
        q, k, v = peaked(torch, tokens, keys, H, Hkv, D, nats, sinks, 0.5, value, seed=keys + D)
        for most in (1, keys):
            o = paged(pkg, torch, q, k, v, "bf16", most)
            bounded(torch, o, q, k, v, "bf16", keys / 4, f"sinks {sinks}, values around {value}")


@pytest.mark.parametrize("D", [64, 128])
def test_prompts_whose_largest_scores_come_late(pkg, torch, D):
    """The reference of a row of the chunk kernel stays while the maximum exceeds it by less than 2^8: keys that grow by a little less and a little more than that, one by one and
    tile by tile."""
    c = scale_of(D)
    for nats, gap in ((0.7, 1), (5.5, 128), (5.6, 128), (11.0, 300)):
        q, k, v = peaked(torch, 200, 1500, 4, 2, D, 0.0, [], 0.3, 40, seed=D)
        levels = ((torch.arange(1500, device="cuda") // gap) * (nats / (c * 127.0))).clamp(max=32 * 127).long()
        for i in range(32):
            k[:, :, i] = (levels // 32 + (i < levels % 32).long()).clamp(max=127).to(torch.int8)[:, None]
        for most in (1, 1500):
            bounded(torch, paged(pkg, torch, q, k, v, "bf16", most), q, k, v, "bf16", 1500 / 4, f"{nats} nats every {gap} keys")


@pytest.mark.parametrize("D,H,tokens", [(128, 3, 1), (64, 7, 1), (64, 16, 1), (128, 8, 20)])
def test_tiny_ranges_of_values_and_many_keys(pkg, torch, D, H, tokens):
    """v_amax = 1e-35: the factor from sums to outputs, v_amax / 127 over a sum of 131,072 keys in units of P, must not fall below what fp32 holds."""
    keys, page = 131072, 64
    q, k, v = peaked(torch, tokens, keys, H, 1, D, 0.0, [], 0.3, 60, seed=H)
    kc, vc = (x.view(keys // page, page, 1, D).transpose(1, 2).contiguous() for x in (k, v))
    o = torch.empty((tokens, H, D), dtype=torch.bfloat16, device="cuda")
    for v_amax in (1e-35, 1e35):
        pkg.FMHAInferI8Paged(None, pkg.FMHAParamI8(AMAX[0], AMAX[1], v_amax, 1.0, 1.0), pkg.AttnDataDescriptorGrouped(1, tokens, keys, H, 1, D), q, kc, vc,
                             torch.arange(keys // page, dtype=torch.int32, device="cuda")[None], torch.tensor([keys], dtype=torch.int32, device="cuda"), starts([tokens]), o)
        s = q.double().transpose(0, 1) @ k[:, 0].double().T * scale_of(D)
        seen = torch.ones((tokens, keys), dtype=torch.bool, device="cuda").tril(keys - tokens)
        want = (torch.softmax(s.masked_fill(~seen, -math.inf), -1) @ v[:, 0].double()).transpose(0, 1) * (float(torch.tensor(v_amax)) / 127.0)
        # all values are positive: half a step of the output, and what bounded() counts for P, exp2 and the sums, all relative
        worst = float(((o.double() - want).abs() / want).max())
        assert worst <= 2.0 ** -8 + 2.0 ** -11 + 2.0 ** -17 + keys / 4 * 2.0 ** -23, (v_amax, worst)


@pytest.mark.parametrize("D,H,Hkv,tokens", [(128, 4, 1, 1), (64, 1, 1, 3), (128, 8, 1, 1), (64, 7, 1, 1), (64, 16, 1, 1), (128, 4, 2, 50), (64, 8, 1, 300)])
def test_the_lowest_code(pkg, torch, D, H, Hkv, tokens):
    """-128, which the quantiser never gives, in q, k and v at once: largest scores, and the largest sums of bytes that a tile can have."""
    keys = 1000
    for q_code, v_code in ((-128, -128), (127, -128), (-128, 127)):
        q = torch.full((tokens, H, D), q_code, dtype=torch.int8, device="cuda")
        k = torch.full((keys, Hkv, D), -128, dtype=torch.int8, device="cuda")
        v = torch.full((keys, Hkv, D), v_code, dtype=torch.int8, device="cuda")
        o = paged(pkg, torch, q, k, v, "fp16", keys)
        bounded(torch, o, q, k, v, "fp16", keys / 4, f"{q_code}, {v_code}")
