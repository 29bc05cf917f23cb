"""CPU tests of the serving kernels' source: no wait's outcome is ignored."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "int8-flash-attention-fmha-quantization_b200", "csrc")


def test_every_way_through_a_tile_asks_whether_its_values_arrived():
    """The wait for V of the rows kernel is asked once and answered in each of the three forms of the product that follow; none may go on without."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "fmha_rows_sm100.cuh")).read())
    assert text.count("mbar_wait_timed(") == 2
    behind = text[text.index("const bool here = mbar_wait_timed(bar_v"):]
    four, eight, sixteen = re.split(r"if constexpr \(kRows == 4\) \{|\} else if constexpr \(kRows == 8\) \{|\n    \} else \{\n", behind)[1:4]
    for form in (four, eight, sixteen):
        first = re.search(r"products\(|mma16816\(", form).start()
        assert "here" in form[:first] and re.search(r"if \(!arrived\(here\)\) break;|if \(!\(ok = __all_sync\(0xFFFFFFFFu, here\)\)\) break;", form[:first])


def test_no_wait_of_the_chunk_kernel_is_ignored():
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "fmha_chunk_sm100.cuh")).read())
    calls = re.findall(r"[^\n;{}]*warp_wait\(", text)
    assert len(calls) > 15
    for call in calls:
        assert "!warp_wait(" in call or "return warp_wait(" in call, call
