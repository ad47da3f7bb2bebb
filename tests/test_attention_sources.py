"""What the attention sources must not hold, by reading them."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gevva_b200", "csrc")


def test_no_read_only_loads():
    """A kernel that is launched while its predecessor runs may not read what that one writes as memory that stays as it is for the whole kernel
    (ld.global.nc, __ldg, pointers that the compiler may take for such)."""
    for name in ("attention.cu", "attention_rows.cu"):
        with open(os.path.join(CSRC, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        assert "launch_chained" in text
        assert not re.search(r"__ldg|\.nc\b|__restrict__", text), name
