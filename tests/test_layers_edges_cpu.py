"""Host side of psgd_pro_b200.layers and its C entries at their edges, without a GPU."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "psgd_pro_b200", "csrc")


def test_every_bounded_launch_takes_the_settable_wait_limit():
    """A kernel's limit comes from wait_limit(), which psgd_set_wait_limit_ns sets: the constant itself is only its default and
    the limit of what an aborting CTA has in flight."""
    given = []
    for name in sorted(os.listdir(CSRC)):
        text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
        assert not re.search(r"wait_ns\s*=\s*WAIT_LIMIT_NS", text), name
        given += re.findall(r"wait_limit\(\)\)|wait_ns = wait_limit\(\)", text)
    assert len(given) >= 4
