"""Rules of the kernels' sources whose breach no result shows: read from the files, without a GPU."""

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "taco_amd", "csrc")


def sources():
    return {n: open(os.path.join(CSRC, n)).read() for n in sorted(os.listdir(CSRC)) if n.endswith((".hip", ".h"))}


def arguments(text, at):
    """The arguments of the call whose opening parenthesis is text[at]."""
    depth, out, start = 0, [], at + 1
    for i in range(at, len(text)):
        depth += (text[i] in "([{") - (text[i] in ")]}")
        if (text[i] == "," and depth == 1) or depth == 0:
            out.append(" ".join(text[start:i].split()))
            start = i + 1
        if depth == 0:
            return out
    raise ValueError("a call without an end")


def buffer_loads(text):
    at = text.find("__builtin_amdgcn_raw_buffer_load")
    while at >= 0:
        yield arguments(text, text.index("(", at))
        at = text.find("__builtin_amdgcn_raw_buffer_load", at + 1)


def test_places_past_a_descriptor_lie_in_the_lanes_offset():
    """A load past the end of its buffer gives zeros without an access where the lane's offset says so; the scalar offset is
    not bounded by that check, so it is 0, or one that the code keeps within the buffer (its end for none)."""
    kept = {"none ? bytes : row * hd"}  # rows below the capacity, `bytes` of which the buffer holds
    seen = 0
    for name, text in sources().items():
        for args in buffer_loads(text):
            seen += 1
            assert args[2] == "0" or args[2] in kept, (name, args)
    assert seen >= 4


def test_tables_are_waited_for():
    """A kernel that copies its table to LDS straight waits for its own loads right before a barrier; the barrier itself waits
    for LDS operations, which these loads are not."""
    there = re.compile(r"\btable_there\(\)|wait_vmcnt<0>\(\);[^\n]*\n\s*(__syncthreads|lds_barrier)\(\)")
    assert there.search(sources()["attend.h"])
    for name, most in (("attend_paged.hip", 4), ("attend_rows.hip", 3)):
        kernels = 0
        for body in re.split(r"\n__global__|\ntemplate <", sources()[name]):
            at = re.search(r"\b(paged|load)_table\((?!const)", body)
            if at:
                kernels += 1
                assert there.search(body, at.end()), body[:200]
                assert not re.search(r"__syncthreads\(\);  // the table", body), body[:200]
        assert kernels == most
