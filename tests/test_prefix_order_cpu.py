"""What the kernels of prefix attention do in front of their first wait for the kernel before them, read from their source."""
import re
from pathlib import Path

SOURCE = re.sub(r"//[^\n]*", "", (Path(__file__).resolve().parent.parent / "llm_b200" / "csrc" / "prefix_attention.cu").read_text())


def kernels():
    """(name, body) of every kernel of the file."""
    for found in re.finditer(r"__global__[^{;]*?\b(\w+_kernel)\(", SOURCE):
        at = start = SOURCE.index("{", found.end())
        depth = 0
        while True:
            depth += {"{": 1, "}": -1}.get(SOURCE[at], 0)
            if depth == 0:
                break
            at += 1
        yield found.group(1), SOURCE[start:at + 1]


def test_no_block_leaves_before_the_kernel_in_front_is_complete():
    """The own parts of a step are launched behind the shared ones' kernel and read what lies in front of both without a wait of their own at their
    start: that a block of the shared ones has left, or has let them start, must say that it has waited."""
    seen = dict(kernels())
    assert len(seen) == 5
    for name, body in seen.items():
        before = body[:re.search(r"(?<!return )griddep_wait\(\);", body).start()]
        leaves = re.findall(r"\breturn\b[^;]*;", before)
        assert all(r == "return griddep_wait();" for r in leaves), (name, leaves)
        if name in ("prefix_attention_tile_kernel", "prefix_attention_wide_kernel"):
            assert "griddep_launch" not in before, name
