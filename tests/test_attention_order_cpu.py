"""CPU: what the attention kernels' source has to hold for their order in tensor memory, since a race there shows in no result for sure."""
import os
import re

import pytest

from htgs_b200 import build

# barriers at which the tensor cores arrive (or, behind a fence of their own, warps that read or wrote tensor memory)
BARRIERS = "scored|summed|graded|added|old|finished|granted"
OBSERVES = re.compile(rf"(?:wait_in_line|mbar_test)\((?:{BARRIERS})\b")
FENCES = re.compile(r"tmem_fence_after\(\)|\bmeet\(\)")                 # `meet` has one behind its wait
TOUCHES = re.compile(r"\b(?:tmem_begin(?:16|32)|tmem_load32|tmem_store(?:16|32)|multiply_seen<T>|store_sums<T>)\(")


def unfenced(text):
    """Lines that touch tensor memory behind a barrier seen to be passed, with no fence between them."""
    found, since = [], None
    for number, line in enumerate(text.splitlines(), 1):
        code = line.split("//")[0]
        if "__global__" in code:
            since = None
        for event in sorted([(m.start(), "seen") for m in OBSERVES.finditer(code)] + [(m.start(), "fence") for m in FENCES.finditer(code)] + [(m.start(), "touch") for m in TOUCHES.finditer(code)]):
            if event[1] == "seen":
                since = number
            elif event[1] == "fence":
                since = None
            elif since is not None:
                found.append((since, number))
    return found


def test_tensor_memory_is_touched_only_behind_a_fence():
    """tcgen05.ld and .st are ordered behind the products that a barrier stands for by tcgen05.fence::after_thread_sync behind the wait or the test that saw it passed, not in front of it."""
    with open(os.path.join(build.CSRC, "attention_tiles.cu")) as f:
        text = f.read()
    assert len(OBSERVES.findall(text)) >= 15 and len(TOUCHES.findall(text)) >= 30
    assert unfenced(text) == []


@pytest.mark.parametrize("text,lines", [("wait_in_line(scored + s, 0, failed);\ntmem_fence_after();\nconst bool used = mbar_test(summed + s, 1);\ntmem_store16(weights, words);", [(3, 4)]),
                                        ("tmem_fence_after();\nif (!free) {\nok = wait_in_line(old, 0, failed);\n}\ntmem_store32(weights, words);", [(3, 5)]),
                                        ("if (!free) {\nok = wait_in_line(old, 0, failed);\ntmem_fence_after();\n}\ntmem_store32(weights, words);", [])])
def test_the_search_finds_what_it_looks_for(text, lines):
    assert unfenced(text) == lines


def test_blocks_with_tensor_memory_that_may_wait_for_one_another_never_share_an_sm():
    """Whoever takes tensor memory asserts, where it is compiled, how much shared memory it has; who takes it ahead of the wait for the kernel before, that it has an SM to itself."""
    ahead = []
    for name in sorted(os.listdir(build.CSRC)):
        if not name.endswith(".cu"):
            continue
        with open(os.path.join(build.CSRC, name)) as f:
            text = f.read()
        kernels = [k for k in re.split(r"(?=\n__global__|\n(?:template <[^\n]*> )__global__)", text) if "__global__" in k and "tcgen05.alloc" in k]
        if not kernels:
            continue
        tiles = re.findall(r"\nstruct (?:\w*Tile|Tile) \{.*?\n\};|> struct \w*Tile \{.*?\n\};", text, re.S)
        assert tiles and all("smem >= kLeastTensorShared" in t for t in tiles), name
        if any(k.index("tcgen05.alloc") < k.index("grid_dependency()") for k in kernels):
            ahead.append(name)
            assert all("alone_with_tensor_memory(smem)" in t for t in tiles), name
    assert ahead == ["fp8_matmul.cu"]
