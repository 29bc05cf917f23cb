"""Performance cases of the serving operators around the INT8 attention: what a program that serves a causal language model with an
int8 cache asks of this package, next to the padded forward passes of cases.py.

  append   rope_quantize_append   rotary positions, quantisation to int8 and the write into the cache's pages, in front of the attention
  prompt   FMHAInferI8Packed      causal attention over whole prompts of different lengths, packed one after the other, grouped heads
  paged    FMHAInferI8Paged       attention of new tokens -- one per sequence, a chunk, or both in one batch -- over a paged int8 cache

Head counts, lengths and value distributions are those of workloads.py (C1: 2 heads of 64, C2: 12 heads of 64 and lengths to 512, C3: 32 heads
of 128 and length 2048, C4: length 16384 and outliers) with grouped key heads, or generic ones between them.  Activations are normal, int8
tensors are quantised symmetrically with a fixed range per tensor, as a calibrated program has it.
"""
import importlib
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "int8": torch.int8}
Q_AMAX, K_AMAX, V_AMAX = 4.5, 4.75, 4.25       # calibrated ranges of normal activations
OUTLIER_GAIN = 8.0


def _package():
    return importlib.import_module("int8-flash-attention-fmha-quantization_b200")


def listed():
    return [
        # the smallest step: the one new token of one request, 12 heads of 64
        dict(name="append_one", kind="append", T=1, H=12, Hkv=12, D=64, rot=64, interleaved=False, dtype="bf16", page=16, scaled=False, first=300),
        # the new tokens of a decoding batch: half of each head rotated, neighbouring elements paired
        dict(name="append_decode", kind="append", T=256, H=32, Hkv=8, D=128, rot=64, interleaved=True, dtype="fp16", page=16, scaled=False, first=4000),
        # a prefill's tokens, far into a long context with scaled frequencies, out of the fused projection's output
        dict(name="append_prompt", kind="append", T=8192, H=32, Hkv=8, D=128, rot=128, interleaved=False, dtype="bf16", page=64, scaled=True, first=98304),
        # the smallest prompt: one short request, two heads (C1): latency of a call
        dict(name="prompt_smallest", kind="prompt", B=1, H=2, Hkv=2, D=64, shortest=64, longest=64, causal=True, out="bf16"),
        # ragged prompts of a batch of requests, three query heads to a key head (C2)
        dict(name="prompt_ragged", kind="prompt", B=32, H=12, Hkv=4, D=64, shortest=1, longest=512, causal=True, out="bf16"),
        # prefill of a batch of equal prompts (C3)
        dict(name="prompt_batch", kind="prompt", B=8, H=32, Hkv=8, D=128, shortest=2048, longest=2048, causal=True, out="bf16"),
        # one long prompt with outliers in Q and K (C4)
        dict(name="prompt_long", kind="prompt", B=1, H=32, Hkv=8, D=128, shortest=16384, longest=16384, causal=True, out="bf16", outliers=0.01),
        # one request's next token
        dict(name="paged_one", kind="paged", B=1, H=32, Hkv=8, D=128, tokens=1, chunks=0, shortest=1025, longest=1025, page=16, out="bf16", tail=0),
        # the next tokens of a batch whose contexts differ widely
        dict(name="paged_decode", kind="paged", B=64, H=32, Hkv=8, D=128, tokens=1, chunks=0, shortest=1, longest=8192, page=16, out="bf16", tail=0),
        # the next tokens of two very long contexts, seven query heads to a key head
        dict(name="paged_decode_long", kind="paged", B=2, H=28, Hkv=4, D=128, tokens=1, chunks=0, shortest=120001, longest=131072, page=64, out="fp16", tail=0),
        # chunks of four prompts over what is cached already, the output quantised for the next projection
        dict(name="paged_chunk", kind="paged", B=4, H=32, Hkv=8, D=128, tokens=500, chunks=4, shortest=6000, longest=8192, page=32, out="int8", tail=0),
        # one chunk of a new prompt in a batch with 32 decoding requests; the buffers are padded to a fixed number of rows
        dict(name="paged_mixed", kind="paged", B=33, H=16, Hkv=2, D=64, tokens=480, chunks=1, shortest=500, longest=4096, page=16, out="bf16", tail=16),
    ]


MOST_SCORES = 2.0e9        # scores of one call over padded sequences, all heads
MOST_CACHE = 1.5e8         # elements of K


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "prompt", "prompt", "paged", "paged", "paged"))
    D = rng.choice((64, 128))
    Hkv = rng.choice((1, 2, 3, 4, 8, 12))
    H = Hkv * rng.choice([g for g in (1, 2, 3, 4, 5, 6, 7, 8, 16) if g * Hkv <= 32])
    if kind == "append":
        T = _log_int(rng, 1, 8192)
        return dict(kind=kind, T=T, H=H, Hkv=Hkv, D=D, rot=rng.choice((D, D // 2, D // 4, 0)), interleaved=rng.random() < 0.5,
                    dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), page=rng.choice((16, 32, 64, 128)), scaled=rng.random() < 0.3,
                    first=rng.randint(0, 100000))
    if kind == "prompt":
        longest = _log_int(rng, 1, 16384)
        B = _log_int(rng, 1, max(1, min(64, int(MOST_SCORES / (H * longest * longest)))))
        return dict(kind=kind, B=B, H=H, Hkv=Hkv, D=D, shortest=rng.randint(1, longest), longest=longest, causal=rng.random() < 0.8,
                    out=rng.choice(("bf16", "bf16", "fp16")))
    longest = _log_int(rng, 2, 131072)
    tokens = 1 if rng.random() < 0.5 else min(longest, _log_int(rng, 2, 2048))
    most_b = min(MOST_CACHE / (Hkv * longest * D), MOST_SCORES / (H * tokens * longest), 128)
    B = _log_int(rng, 1, max(1, int(most_b)))
    chunks = 0 if tokens == 1 else B if rng.random() < 0.6 else rng.randint(1, B)
    return dict(kind=kind, B=B, H=H, Hkv=Hkv, D=D, tokens=tokens, chunks=chunks, shortest=rng.randint(tokens, longest), longest=longest,
                page=rng.choice((16, 32, 64, 128)), out=rng.choice(("bf16", "bf16", "fp16")), tail=rng.choice((0, 0, 7)))


def _lengths(case):
    """Keys of each sequence, from the case alone: any number between the shortest and the longest."""
    r = random.Random("%d %d %d" % (case["B"], case["shortest"], case["longest"]))
    return [r.randint(case["shortest"], case["longest"]) for _ in range(case["B"])]


def _new_tokens(case):
    """Query rows of each sequence: one, or a chunk in the last ones."""
    if case["kind"] == "prompt":
        return _lengths(case)
    return [1] * (case["B"] - case["chunks"]) + [case["tokens"]] * case["chunks"]


def _generator(seed, k):
    g = torch.Generator(device="cuda")
    g.manual_seed(16 * seed + k)
    return g


def _codes(shape, amax, outliers, g):
    """Normal values in int8 codes of the range [-amax, amax]; outliers widen the range by what they are larger."""
    x = torch.randn(shape, generator=g, device="cuda")
    if outliers:
        x = torch.where(torch.rand(shape, generator=g, device="cuda") < outliers, x * OUTLIER_GAIN, x)
    return x.mul_(127.0 / amax).round_().clamp_(-127, 127).to(torch.int8)


def _starts(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _inv_freq(case):
    """Angles per position of the pairs of a head.  Scaled: frequencies with more than 32 turns in 4096 positions stay, those with less than one
    are slowed down 16 times, those between partly, and the magnitude grows by 0.1 ln 16."""
    half = case["rot"] // 2
    f = [500000.0 ** (-2.0 * i / case["rot"]) for i in range(half)] if half else []
    if not case["scaled"]:
        return f, 1.0
    turns = [4096.0 * w / (2 * math.pi) for w in f]
    keep = [min(1.0, max(0.0, (t - 1.0) / 31.0)) for t in turns]
    return [w * (k + (1.0 - k) / 16.0) for w, k in zip(f, keep)], 0.1 * math.log(16.0) + 1.0


def prepare(case, seed):
    D, H, Hkv = case["D"], case["H"], case["Hkv"]
    if case["kind"] == "append":
        T, page, rot = case["T"], case["page"], case["rot"]
        qkv = torch.randn((T, H + 2 * Hkv, D), generator=_generator(seed, 0), device="cuda").to(TYPES[case["dtype"]])
        pages = -(-(T + page) // page)
        cache = torch.zeros((2, pages, Hkv, page, D), dtype=torch.int8, device="cuda")
        slots = torch.randperm(pages * page, generator=_generator(seed, 1), device="cuda")[:T].contiguous()
        if T >= 64:
            slots[5] = -1                       # a padded row: nothing is stored for it
        inv_freq, magnitude = _inv_freq(case)
        s = dict(case=case, q=qkv[:, :H], k=qkv[:, H:H + Hkv], v=qkv[:, H + Hkv:], slots=slots, k_cache=cache[0], v_cache=cache[1],
                 q_out=torch.empty((T, H, D), dtype=torch.int8, device="cuda"),
                 positions=torch.arange(case["first"], case["first"] + T, dtype=torch.int32, device="cuda"),
                 inv_freq=torch.tensor(inv_freq, dtype=torch.float64, device="cuda"), magnitude=magnitude)
        # The table that a program makes once for its model: cosine and sine of every pair at every position, a 32-bit value and, in a
        # second plane, what that leaves of the 64-bit one.
        angle = torch.arange(case["first"] + T, device="cuda").double()[:, None] * s["inv_freq"]
        turns = torch.stack((torch.cos(angle), torch.sin(angle)), -1).flatten(1) * magnitude
        s["table"] = torch.stack((turns.float(), (turns - turns.float().double()).float()))
        if own:
            s["pkg"] = pkg = _package()
            s["param"] = pkg.FMHAParamI8(Q_AMAX, K_AMAX, V_AMAX, 1.0, 1.0)
        return s
    lengths, new = _lengths(case), _new_tokens(case)
    outliers = case.get("outliers", 0.0)
    amax_q, amax_k = (a * (OUTLIER_GAIN if outliers else 1.0) for a in (Q_AMAX, K_AMAX))
    rows = sum(new) + case.get("tail", 0)
    # the calibrated range of the output: six standard deviations of an average over the shortest context
    o_amax = min(V_AMAX, 6.0 * math.sqrt(min(1.0, math.exp(1.0) / case["shortest"])))
    s = dict(case=case, q=_codes((rows, H, D), amax_q, outliers, _generator(seed, 0)), cu_q=_starts(new), max_q=max(new), max_k=max(lengths),
             amax=(amax_q, amax_k, V_AMAX, o_amax), o=torch.zeros((rows, H, D), dtype=TYPES[case["out"]], device="cuda"), causal=case.get("causal", True))
    if case["kind"] == "prompt":
        s["k"] = _codes((rows, Hkv, D), amax_k, outliers, _generator(seed, 1))
        s["v"] = _codes((rows, Hkv, D), V_AMAX, 0.0, _generator(seed, 2))
        s["cu_k"] = s["cu_q"]
    else:
        page = case["page"]
        wanted = [-(-n // page) for n in lengths]
        pages = sum(wanted) + 3
        order = torch.randperm(pages, generator=_generator(seed, 3), device="cuda").to(torch.int32).cpu()
        table, at = torch.zeros((case["B"], max(wanted)), dtype=torch.int32), 0
        for b, n in enumerate(wanted):
            table[b, :n] = order[at:at + n]
            at += n
        s["k"] = _codes((pages, Hkv, page, D), amax_k, outliers, _generator(seed, 1))
        s["v"] = _codes((pages, Hkv, page, D), V_AMAX, 0.0, _generator(seed, 2))
        s["page_table"] = table.cuda()
        s["seqlens_k"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    if own:
        s["pkg"] = pkg = _package()
        s["param"] = pkg.FMHAParamI8(*s["amax"], 1.0)
        s["desc"] = pkg.AttnDataDescriptorGrouped(case["B"], s["max_q"], s["max_k"], H, Hkv, D)
    return s


def run(s):
    case = s["case"]
    if case["kind"] == "append":
        if own:
            s["pkg"].rope_quantize_append(None, s["param"], s["q"], s["k"], s["v"], s["positions"], s["table"], s["q_out"], s["k_cache"], s["v_cache"],
                                          slots=s["slots"], interleaved=case["interleaved"])
        else:
            _plain_append(s)
        # the codes themselves: they are the exact ones, a value next to a border is decided in 64 bits
        return s["q_out"], s["k_cache"], s["v_cache"]
    if own:
        if case["kind"] == "prompt":
            s["pkg"].FMHAInferI8Packed(None, s["param"], s["desc"], s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], s["o"], causal=s["causal"])
        else:
            s["pkg"].FMHAInferI8Paged(None, s["param"], s["desc"], s["q"], s["k"], s["v"], s["page_table"], s["seqlens_k"], s["cu_q"], s["o"],
                                      causal=s["causal"])
    else:
        _plain_attention(s)
    if case["out"] == "int8":
        return s["o"].to(torch.bfloat16).mul_(s["amax"][3] / 127.0)       # the values that the codes stand for
    return s["o"]


def _plain_append(s):
    case = s["case"]
    rot = case["rot"]
    turns = s["table"][:, s["positions"].long()].double().sum(0)[:, None]
    cos, sin = turns[..., 0::2], turns[..., 1::2]

    def rotate(x):
        y = x.double()
        if rot:
            a, b = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
            x1, x2 = y[..., a].clone(), y[..., b].clone()
            y[..., a] = x1 * cos - x2 * sin
            y[..., b] = x2 * cos + x1 * sin
        return y

    def quantise(y, amax):
        return torch.floor(y * (127.0 / amax) + 0.5).clamp(-127, 127).to(torch.int8)

    s["q_out"].copy_(quantise(rotate(s["q"]), Q_AMAX))
    stored = s["slots"] >= 0
    slots = s["slots"][stored]
    page, at = slots // case["page"], slots % case["page"]
    s["k_cache"][page, :, at] = quantise(rotate(s["k"]), K_AMAX)[stored]
    s["v_cache"][page, :, at] = quantise(s["v"].double(), V_AMAX)[stored]


def _plain_attention(s):
    """All sequences padded to the longest, in 32 bits."""
    case = s["case"]
    D, H, Hkv = case["D"], case["H"], case["Hkv"]
    G, B = H // Hkv, case["B"]
    q_amax, k_amax, v_amax, o_amax = s["amax"]
    cu_q = s["cu_q"].long()
    len_q = cu_q[1:] - cu_q[:-1]
    i, j = torch.arange(s["max_q"], device="cuda"), torch.arange(s["max_k"], device="cuda")
    if case["kind"] == "prompt":
        cu_k = s["cu_k"].long()
        len_k = cu_k[1:] - cu_k[:-1]
        at = (cu_k[:-1, None] + j).clamp(max=s["k"].shape[0] - 1)
        k, v = (x[at].transpose(1, 2).float() for x in (s["k"], s["v"]))                       # [B, Hkv, max_k, D]
    else:
        len_k = s["seqlens_k"].long()
        pages = s["page_table"].long()[:, j // case["page"]]
        k, v = (x[pages, :, j % case["page"]].transpose(1, 2).float() for x in (s["k"], s["v"]))
    rows = (cu_q[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].view(B, s["max_q"], Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * s["max_q"], D).float()
    scores = torch.matmul(q, k.transpose(2, 3))
    scores *= q_amax * k_amax / (127.0 * 127.0 * math.sqrt(D))
    seen = j < len_k[:, None, None]
    if s["causal"]:
        seen = seen & (j <= (i + (len_k - len_q)[:, None])[:, :, None])
    scores.view(B, Hkv, G, s["max_q"], s["max_k"]).masked_fill_(~seen[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True).clamp(min=-1e30)
    p = scores.exp_()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-30) * (v_amax / 127.0)
    o = o.view(B, Hkv, G, s["max_q"], D).permute(0, 3, 1, 2, 4).reshape(B, s["max_q"], H, D)
    real = i < len_q[:, None]
    if case["out"] == "int8":
        o = (o * (127.0 / o_amax)).round().clamp(-127, 127)
    s["o"][rows[real]] = o[real].to(s["o"].dtype)


def work(case):
    D, H, Hkv = case["D"], case["H"], case["Hkv"]
    if case["kind"] == "append":
        T, size = case["T"], TYPES[case["dtype"]].itemsize
        elements = T * (H + 2 * Hkv) * D
        # in, the cosines and sines of its positions, slots and positions, out
        return {"bytes": elements * (size + 1.0) + T * (4.0 * case["rot"] + 12), "flops": elements * 5.0}
    lengths, new = _lengths(case), _new_tokens(case)
    if case.get("causal", True):
        pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, lengths))
    else:
        pairs = sum(n * m for n, m in zip(new, lengths))
    return {"bytes": sum(new) * H * D * (1.0 + TYPES[case["out"]].itemsize) + 2.0 * sum(lengths) * Hkv * D, "flops": 4.0 * H * D * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    D, H, Hkv = case["D"], case["H"], case["Hkv"]
    if case["kind"] == "append":
        return _exact_append(s)
    if case["out"] == "int8":
        return None          # an output next to a border of two codes has two neighbours, and either is right
    cu_q = s["cu_q"].tolist()
    o = torch.zeros((s["q"].shape[0], H, D), dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        first, last = cu_q[b], cu_q[b + 1]
        if case["kind"] == "prompt":
            k, v = s["k"][first:last], s["v"][first:last]
        else:
            pages = s["page_table"][b, :-(-n // case["page"])].long()
            k, v = (x[pages].permute(0, 2, 1, 3).reshape(-1, Hkv, D)[:n] for x in (s["k"], s["v"]))
        visible = torch.ones((last - first, n), dtype=torch.bool, device="cuda")
        if s["causal"]:
            visible = visible.tril(n - (last - first))
        for h in range(H):
            x = s["q"][first:last, h].double() * (s["amax"][0] / 127.0)
            y, z = (t[:, h // (H // Hkv)].double() for t in (k, v))
            logits = (x @ (y * (s["amax"][1] / 127.0)).T).div_(math.sqrt(D)).masked_fill_(~visible, -math.inf)
            weights = torch.exp(logits - torch.logsumexp(logits, 1, keepdim=True))
            o[first:last, h] = weights @ (z * (s["amax"][2] / 127.0))
    return o


def _exact_append(s):
    """Pairs as complex numbers, turned by e^(i angle)."""
    case = s["case"]
    rot = case["rot"]
    angle = torch.outer(s["positions"].double(), s["inv_freq"])
    turn = torch.polar(torch.full_like(angle, s["magnitude"]), angle).unsqueeze(1)

    def code(x, amax, rotated):
        x = x.to(torch.float64)
        if rotated and rot:
            head, rest = x[..., :rot], x[..., rot:]
            if case["interleaved"]:
                z = torch.view_as_complex(head.reshape(*head.shape[:-1], rot // 2, 2).contiguous()) * turn
                head = torch.view_as_real(z).flatten(-2)
            else:
                z = torch.complex(head[..., :rot // 2].contiguous(), head[..., rot // 2:].contiguous()) * turn
                head = torch.cat((z.real, z.imag), -1)
            x = torch.cat((head, rest), -1)
        return torch.clamp(torch.floor(x * (127.0 / amax) + 0.5), -127.0, 127.0).to(torch.int8)

    k, v = torch.zeros_like(s["k_cache"]), torch.zeros_like(s["v_cache"])
    for x, cache, amax, rotated in ((s["k"], k, K_AMAX, True), (s["v"], v, V_AMAX, False)):
        flat = cache.transpose(1, 2).reshape(-1, case["Hkv"], case["D"])         # one row per slot
        kept = s["slots"] >= 0
        flat[s["slots"][kept]] = code(x, amax, rotated)[kept]
        cache.copy_(flat.view(cache.shape[0], case["page"], case["Hkv"], case["D"]).transpose(1, 2))
    return code(s["q"], Q_AMAX, True), k, v
