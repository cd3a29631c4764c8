"""Newton-Schulz products on the host: what the kernels' source, the library's own choices and the entry points' arguments have to hold, without a GPU."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "mini_trainer_b200" / "csrc"


def body(source, name):
    """Text of a function, without its comments."""
    source = re.sub(r"//[^\n]*", "", source)
    at = source.index("{", source.index(") {", re.search(rf"\b{name}\(const", source).start()))
    depth = 0
    for i in range(at, len(source)):
        depth += {"{": 1, "}": -1}.get(source[i], 0)
        if depth == 0:
            return source[at:i]


@pytest.mark.parametrize("name", ["product_kernel", "split_kernel", "small_kernel"])
def test_warps_are_whole_before_aligned_instructions(name):
    """An instruction that is .aligned (allocation and loads of tensor memory, barriers of a cluster) is for warps whose threads come to it together, which nothing promises behind a block of one thread or
    a wait that each thread ends by itself: a barrier of the warp or the block has to be between."""
    together = r"__all_sync\(0xffffffffu, mbar_wait\(|__syncwarp\(\)|__syncthreads\(\)"
    apart = r"threadIdx\.x == 0\)|lane == 0\)|elect_one\(\)|mbar_wait\(|wait_sent\("
    aligned = r"cluster_barrier\(\)|tmem_alloc\(|tcgen05\.alloc|tmem_ld_\w+\(|tmem_dealloc\(|tcgen05\.dealloc"
    text, whole, seen = body((CSRC / "newton_schulz.cu").read_text(), name), True, 0
    for m in re.finditer(f"(?P<together>{together})|(?P<apart>{apart})|(?P<aligned>{aligned})", text):
        if m.lastgroup == "aligned":
            seen += 1
            assert whole, f"{name}: {text[max(0, m.start() - 300):m.end()]}"
        else:
            whole = m.lastgroup == "together"
    assert seen >= 5
