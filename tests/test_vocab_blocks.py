"""Launches at a language model's two ends that may start early count on a number of blocks on every SM: each kernel says how many it
leaves registers for, so that this does not hang on a compiler's choice."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "katsu_b200" / "csrc"


def kernels(text):
    """(name, arguments of its launch bounds) of every kernel."""
    found = []
    for m in re.finditer(r"__global__ void __launch_bounds__\(", text):
        depth, end, commas = 1, m.end(), 0
        while depth:
            depth += {"(": 1, ")": -1}.get(text[end], 0)
            commas += text[end] == "," and depth == 1
            end += 1
        found.append((re.match(r"\s*(\w+)\(", text[end:]).group(1), commas + 1))
    return found


@pytest.mark.parametrize("name", ["embed.cu", "distill.cu", "logits.cu"])
def test_kernels_say_how_many_of_their_blocks_fit(name):
    text = (CSRC / name).read_text()
    found = kernels(text)
    assert len(found) == text.count("__global__") and found
    assert [kernel for kernel, arguments in found if arguments != 2] == []
