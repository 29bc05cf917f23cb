"""CPU tests of the serving calls' refusals: the C ABI with addresses that are never read, and the Python calls with CPU tensors."""
import ctypes
import os
import re

import pytest
import torch

from _serving import AMAX

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def ll(*x):
    return (ctypes.c_longlong * len(x))(*x)


def packed(pkg, desc=(2, 10, 10, 4, 2, 64), amax=(1, 1, 1, 1, 1), ptrs=(256, 512, 768, 1024, 1280, 2048), o_type=1, tokens=(20, 20), strides=(256, 128, 128, 256), flags=5):
    vp = [ctypes.c_void_p(p) if p else None for p in ptrs]
    return pkg.lib().fmha_i8_sm100_infer_packed(None, (ctypes.c_float * 5)(*amax), (ctypes.c_int * 6)(*desc), *vp, o_type, ll(*tokens), ll(*strides), flags)


def paged(pkg, desc=(2, 1, 100, 4, 2, 64), amax=(1, 1, 1, 1, 1), ptrs=(256, 512, 768, 1024, 1280, 1536, 2048), o_type=1, tokens=2, strides=(256, 256),
          cache=(8, 16, 2048, 4, 4), flags=5):
    vp = [ctypes.c_void_p(p) if p else None for p in ptrs]
    return pkg.lib().fmha_i8_sm100_infer_paged(None, (ctypes.c_float * 5)(*amax), (ctypes.c_int * 6)(*desc), *vp, o_type, tokens, ll(*strides), ll(*cache), flags)


def append(pkg, dims=(4, 4, 2, 64, 64), amax=(1, 1, 1, 1, 1), q=256, k=512, v=768, in_type=1, strides=(256, 128, 128), positions=1024, table=2048, in_table=10,
           outs=(256, 512, 768), slots=1280, cache=(8, 16, 2048)):
    vp = lambda p: ctypes.c_void_p(p) if p else None  # noqa: E731
    return pkg.lib().fmha_i8_sm100_rope_quantize_append(None, (ctypes.c_float * 5)(*amax), ll(*dims), vp(q), vp(k), vp(v), in_type, ll(*strides), vp(positions), vp(table),
                                                        in_table, 0, *[vp(x) for x in outs], vp(slots), ll(*cache) if cache else None)


def test_packed_refusals(pkg):
    for i in range(6):
        ptrs = [256, 512, 768, 1024, 1280, 2048]
        ptrs[i] = 0
        assert packed(pkg, ptrs=ptrs) == pkg.ERR_NULL_POINTER
    assert packed(pkg, flags=4) == pkg.ERR_NO_CUDA_CORE_PATH
    assert packed(pkg, flags=1 | 2) == pkg.ERR_BAD_FLAGS and packed(pkg, flags=1 | 8) == pkg.ERR_BAD_FLAGS
    for desc in ((0, 10, 10, 4, 2, 64), (2, -1, 10, 4, 2, 64), (2, 10, -1, 4, 2, 64), (2, 10, 10, 4, 3, 64), (2, 10, 10, 0, 2, 64), (2, 10, 10, 4, 0, 64),
                 (2, 10, 10, 4, 2, 96)):
        assert packed(pkg, desc=desc) == pkg.ERR_BAD_SHAPE, desc
    assert packed(pkg, o_type=3) == pkg.ERR_BAD_SHAPE
    assert packed(pkg, tokens=(-1, 20)) == pkg.ERR_BAD_SHAPE and packed(pkg, tokens=(20, -1)) == pkg.ERR_BAD_SHAPE
    for strides in ((255, 128, 128, 256), (256, 127, 128, 256), (256, 128, 112, 256), (256, 128, 128, 255)):
        assert packed(pkg, strides=strides) == pkg.ERR_BAD_SHAPE, strides
    for strides in ((264, 128, 128, 256), (256, 136, 128, 256), (256, 128, 136, 256), (256, 128, 128, 260)):
        assert packed(pkg, strides=strides) == pkg.ERR_MISALIGNED, strides
    for i, bad in ((0, 264), (1, 520), (2, 776), (3, 1026), (4, 1282), (5, 2056)):
        ptrs = [256, 512, 768, 1024, 1280, 2048]
        ptrs[i] = bad
        assert packed(pkg, ptrs=ptrs) == pkg.ERR_MISALIGNED, i
    for amax in ((0, 1, 1, 1, 1), (1, float("inf"), 1, 1, 1), (1, 1, float("nan"), 1, 1)):
        assert packed(pkg, amax=amax) == pkg.ERR_BAD_AMAX
    assert packed(pkg, o_type=0, strides=(256, 128, 128, 256), amax=(1, 1, 1, 0, 1)) == pkg.ERR_BAD_AMAX
    assert packed(pkg, tokens=(1 << 30, 20)) == pkg.ERR_TOO_LARGE and packed(pkg, tokens=(20, (1 << 30) + 1)) == pkg.ERR_TOO_LARGE
    assert packed(pkg, desc=(2, 10, (1 << 30) + 1, 4, 2, 64)) == pkg.ERR_TOO_LARGE
    assert pkg.lib().fmha_i8_sm100_last_status() == pkg.ERR_TOO_LARGE


def test_paged_refusals(pkg):
    for i in range(7):
        ptrs = [256, 512, 768, 1024, 1280, 1536, 2048]
        ptrs[i] = 0
        assert paged(pkg, ptrs=ptrs) == pkg.ERR_NULL_POINTER
    for cache in ((0, 16, 2048, 4, 4), (8, 8, 2048, 4, 4), (8, 24, 4096, 4, 4), (8, 8192, 1 << 24, 4, 4), (8, 16, 2032, 4, 4), (8, 16, 2048, 0, 4), (8, 16, 2048, 4, 3)):
        assert paged(pkg, cache=cache) == pkg.ERR_BAD_SHAPE, cache
    assert paged(pkg, cache=(8, 16, 2056, 4, 4)) == pkg.ERR_MISALIGNED
    assert paged(pkg, cache=(8, 16, 2048, 1 << 27, 1 << 27)) == pkg.ERR_TOO_LARGE
    assert paged(pkg, cache=(0x7FFFFFFF, 16, 2048, 4, 4)) == pkg.ERR_TOO_LARGE
    assert paged(pkg, desc=(2, 1, 100, 5, 2, 64)) == pkg.ERR_BAD_SHAPE
    assert paged(pkg, flags=0) == pkg.ERR_NO_CUDA_CORE_PATH


def test_append_refusals(pkg):
    for name in ("q", "k", "v", "positions", "table"):
        assert append(pkg, **{name: 0}) == pkg.ERR_NULL_POINTER, name
    assert append(pkg, outs=(0, 512, 768)) == pkg.ERR_NULL_POINTER and append(pkg, cache=None) == pkg.ERR_NULL_POINTER
    for dims in ((-1, 4, 2, 64, 64), (4, 0, 2, 64, 64), (4, 4, 0, 64, 64), (4, 4, 2, 80, 64), (4, 4, 2, 64, 8), (4, 4, 2, 64, 80), (4, 4, 2, 64, -16)):
        assert append(pkg, dims=dims) == pkg.ERR_BAD_SHAPE, dims
    assert append(pkg, in_type=0) == pkg.ERR_BAD_SHAPE and append(pkg, in_type=4) == pkg.ERR_BAD_SHAPE
    assert append(pkg, strides=(255, 128, 128)) == pkg.ERR_BAD_SHAPE and append(pkg, strides=(260, 128, 128)) == pkg.ERR_MISALIGNED
    assert append(pkg, q=264) == pkg.ERR_MISALIGNED and append(pkg, slots=1284) == pkg.ERR_MISALIGNED and append(pkg, outs=(256, 520, 768)) == pkg.ERR_MISALIGNED
    assert append(pkg, cache=(8, 12, 2048)) == pkg.ERR_BAD_SHAPE and append(pkg, cache=(8, 16, 2032)) == pkg.ERR_BAD_SHAPE
    assert append(pkg, amax=(1, 1, -1, 1, 1)) == pkg.ERR_BAD_AMAX and append(pkg, amax=(1e-38, 1, 1, 1, 1)) == pkg.ERR_BAD_AMAX
    assert append(pkg, dims=(1 << 30, 4, 2, 64, 64)) == pkg.ERR_TOO_LARGE
    L = pkg.lib()
    vp = ctypes.c_void_p
    assert L.fmha_i8_sm100_rope_table(None, None, 4, 10, 1.0, vp(256)) == pkg.ERR_NULL_POINTER
    assert L.fmha_i8_sm100_rope_table(None, vp(256), 0, 10, 1.0, vp(256)) == pkg.ERR_BAD_SHAPE
    assert L.fmha_i8_sm100_rope_table(None, vp(256), 65, 10, 1.0, vp(256)) == pkg.ERR_BAD_SHAPE
    assert L.fmha_i8_sm100_rope_table(None, vp(256), 4, 10, float("nan"), vp(256)) == pkg.ERR_BAD_AMAX
    assert L.fmha_i8_sm100_rope_table(None, vp(260), 4, 10, 1.0, vp(256)) == pkg.ERR_MISALIGNED


def _packed_tensors():
    i8 = lambda *s: torch.zeros(s, dtype=torch.int8)  # noqa: E731
    return dict(q=i8(20, 4, 64), k=i8(20, 2, 64), v=i8(20, 2, 64), cu_seqlens_q=torch.zeros(3, dtype=torch.int32), cu_seqlens_k=torch.zeros(3, dtype=torch.int32),
                o=torch.zeros((20, 4, 64), dtype=torch.bfloat16))


def test_python_packed_checks_its_tensors(pkg):
    param, desc = pkg.FMHAParamI8(*AMAX, 1.0, 1.0), pkg.AttnDataDescriptorGrouped(2, 10, 10, 4, 2, 64)

    def call(**change):
        pkg.FMHAInferI8Packed(0, param, desc, **{**_packed_tensors(), **change})

    with pytest.raises(ValueError, match="not a CUDA tensor"):
        call()
    i8 = lambda *s: torch.zeros(s, dtype=torch.int8)  # noqa: E731
    for name, x in (("q", i8(20, 4, 128)), ("q", i8(20, 4, 64, 1)), ("q", i8(20, 4, 64).float()), ("k", i8(20, 4, 64)), ("v", i8(19, 2, 64)), ("o", torch.zeros(20, 4, 64)),
                    ("o", torch.zeros((19, 4, 64), dtype=torch.bfloat16)), ("cu_seqlens_q", torch.zeros(2, dtype=torch.int32)),
                    ("cu_seqlens_k", torch.zeros(3, dtype=torch.int64)), ("q", i8(4, 20, 64).transpose(0, 1)), ("k", i8(20, 2, 128)[..., ::2]),
                    ("cu_seqlens_q", torch.zeros(6, dtype=torch.int32)[::2])):
        with pytest.raises(ValueError, match=name):
            call(**{name: x})
    with pytest.raises(TypeError, match="torch tensor"):
        call(q=256)


def test_python_paged_and_append_check_their_tensors(pkg):
    param, desc = pkg.FMHAParamI8(*AMAX, 1.0, 1.0), pkg.AttnDataDescriptorGrouped(2, 1, 64, 4, 2, 64)
    i8 = lambda *s: torch.zeros(s, dtype=torch.int8)  # noqa: E731
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    good = dict(q=i8(2, 4, 64), k_cache=i8(8, 2, 16, 64), v_cache=i8(8, 2, 16, 64), page_table=i32(2, 4), seqlens_k=i32(2), cu_seqlens_q=i32(3), o=i8(2, 4, 64))
    with pytest.raises(ValueError, match="not a CUDA tensor"):
        pkg.FMHAInferI8Paged(0, param, desc, **good)
    for name, x in (("k_cache", i8(8, 16, 2, 64)), ("v_cache", i8(8, 2, 32, 64)), ("v_cache", i8(8, 4, 16, 64)[:, :2]), ("page_table", i32(3, 4)), ("seqlens_k", i32(3)),
                    ("page_table", i32(2, 8)[:, ::2]), ("cu_seqlens_q", i32(2)), ("k_cache", i8(8, 16, 2, 64).transpose(1, 2))):
        with pytest.raises(ValueError, match=name):
            pkg.FMHAInferI8Paged(0, param, desc, **{**good, name: x})
    b = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    good = dict(q=b(3, 4, 64), k=b(3, 2, 64), v=b(3, 2, 64), positions=i32(3), table=torch.zeros(2, 9, 64), q_out=i8(3, 4, 64), k_out=i8(8, 2, 16, 64), v_out=i8(8, 2, 16, 64),
                slots=torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="not a CUDA tensor"):
        pkg.rope_quantize_append(0, param, **good)
    for name, x in (("k", b(2, 2, 64)), ("v", b(3, 2, 64).half()), ("positions", i32(4)), ("positions", torch.zeros(3, dtype=torch.int64)), ("table", torch.zeros(9, 64)),
                    ("q_out", i8(3, 2, 64)), ("k_out", i8(3, 2, 64)), ("slots", i32(3)), ("q_out", i8(3, 8, 64)[:, ::2])):
        with pytest.raises(ValueError, match=name):
            pkg.rope_quantize_append(0, param, **{**good, name: x})
    with pytest.raises(ValueError, match="k_out"):
        pkg.rope_quantize_append(0, param, **{**good, "slots": None})


def test_the_serving_kernels_use_ordinary_loads():
    """They start while the kernel before them may still be writing (follow_previous_kernel): no load may be declared read-only."""
    csrc = os.path.join(ROOT, "int8-flash-attention-fmha-quantization_b200", "csrc")
    seen = 0
    for name in sorted(os.listdir(csrc)):
        text = re.sub(r"//[^\n]*", "", open(os.path.join(csrc, name)).read())
        if "follow_previous_kernel();" in text:
            seen += 1
            assert "__ldg" not in text and "__restrict__" not in text, name
    assert seen >= 2
