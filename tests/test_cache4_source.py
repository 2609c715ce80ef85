"""What the source of the 4-bit cache's attention has to say wherever it is compiled: instructions that are a whole warp's
(tcgen05.ld, tcgen05.st, the cluster barrier's .aligned forms) never stand behind something that single lanes did - a wait that each
lane leaves by itself, an arrival of one lane, a branch of some - without a __syncwarp between. What a compiler makes of a source without
it may run for years and then end in a fault, so this is read from the source, not tried."""
import os
import re

import pytest

import helpers as H

CSRC = os.path.join(H.ROOT, "brisk_llm_b200", "csrc")
# lanes part: a wait of each lane's own, or a branch that only some of a warp's lanes take
PARTS = re.compile(r"\bmbar_wait\(|\bmbar_drain\(|\bif \([^;{]*\b(lane|real|leader|tid & 127|tid < k\w+|x < kRows)\b")
WHOLE = re.compile(r"__syncwarp\(\)|\bmbar_wait_warp\(|__syncthreads\(\)")
ALIGNED = re.compile(r"\b(tmem_ld\w*|tmem_st\w*|result_of|scale_columns|add_up|more_registers|fewer_registers|mma16816|transposed)\s*[(<]|\.sync\.aligned|\.aligned;")


def statements(name):
    """The file's lines without comments, and each loop's body once more behind it (its first lines follow its last)."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    lines = list(enumerate(text.split("\n"), 1))
    out, opened = [], []
    for number, line in lines:
        out.append((number, line))
        indent = len(line) - len(line.lstrip())
        if re.match(r"\s*for \(.*\{\s*$", line):
            opened.append((indent, len(out)))
        elif line.strip() == "}" and opened and opened[-1][0] == indent:
            _, begin = opened.pop()
            out.extend(out[begin:])
    return out


@pytest.mark.parametrize("name", ["cache4_prompt.cu", "cache4_attn.cu"])
def test_a_warp_is_whole_where_an_instruction_is_a_whole_warp_s(name):
    apart, wrong = None, set()
    for number, line in statements(name):
        if "__device__ __forceinline__" in line or "__global__" in line or line.startswith("    } else"):
            apart = None  # a function's caller is looked at where it calls; other warps' part of a kernel begins with them whole
        if WHOLE.search(line):
            apart = None
        elif ALIGNED.search(line):
            if apart is not None:
                wrong.add((apart, number))
        elif PARTS.search(line):
            apart = number
    assert not wrong, sorted(wrong)


@pytest.mark.parametrize("name", ["cache4_prompt.cu", "cache4_attn.cu"])
def test_warps_meet_whole_at_the_cluster_s_barrier(name):
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    met = [text.rindex("void ", 0, x.start()) for x in re.finditer(r"barrier\.cluster\.(arrive|wait)", text)]
    assert met
    for begin in met:
        body = text[begin:text.index("barrier.cluster", begin)]
        assert "__syncwarp();" in body, body


def test_the_waits_of_the_many_rows_kernel_are_a_warp_s():
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "cache4_prompt.cu")).read())
    assert not re.search(r"\bmbar_wait\(", text) and len(re.findall(r"\bmbar_wait_warp\(", text)) >= 6
    helper = open(os.path.join(CSRC, "tc.cuh")).read().split("void mbar_wait_warp(")[1].split("\n}")[0]
    assert helper.index("mbar_wait(") < helper.index("__any_sync") < helper.index("__syncwarp();")


def test_what_the_converters_saw_is_read_behind_their_own_barrier():
    """The softmax's warps ask whether a scale was past_f16 behind a wait for the last values, on which the converters arrive after they wrote it."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "cache4_prompt.cu")).read())
    write, arrive = text.index("bar->large = 1"), text.index("mbar_arrive(&bar->v_full[slot])")
    wait, read = text.index("mbar_wait_warp(&bar->v_full[(tiles - 1) & 1]"), text.index("*large != 0")
    assert write < arrive and wait < read
