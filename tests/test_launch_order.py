"""The order that launch.h asks of kernels which start under the one before them, read off their sources: a kernel lets the next one
start after its own wait, so that no more than two overlap and the record of the last launch's outputs is enough."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tessera_b200", "csrc")


def kernels():
    """(name, text without comments) of every kernel, up to the next one."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        with open(path) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for part in text.split("__global__")[1:]:
            yield os.path.basename(path) + ":" + re.search(r"(\w+_kernel)\(", part).group(1), part


def test_a_kernel_waits_before_it_lets_the_next_one_start():
    found = dict(kernels())
    assert len(found) > 30
    triggers = [name for name, text in found.items() if "pdl_trigger()" in text]
    assert len(triggers) >= 8
    early = [name for name in triggers if not 0 <= found[name].find("pdl_wait()") < found[name].find("pdl_trigger()")]
    assert early == []
