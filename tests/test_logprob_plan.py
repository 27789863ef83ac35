"""How many CTAs a row of log probabilities gets (tessera_b200/csrc/logprob_plan.h), compiled by the host compiler."""
import os
import subprocess

import pytest

from test_attention_plan import DEVICES, ROOT


@pytest.mark.parametrize("resident", DEVICES)
def test_clusters_of_a_row(tmp_path, resident):
    """As many as the machine has room for and the vocabulary has work for, of the sizes that the device takes."""
    cases = [(r, v) for r in (1, 9, 10, 16, 18, 19, 37, 38, 148, 149, 65535) for v in (1, 3000, 3100, 12288, 24575, 24576, 151936, 2**31 - 10000)]
    fits = "[](unsigned c) { return c == 1 ? %d : c == 2 ? %d : c == 4 ? %d : c == 8 ? %d : %d; }" % tuple(resident[c] for c in (1, 2, 4, 8, 16))
    (tmp_path / "p.cpp").write_text('#include <cstdio>\n#include "logprob_plan.h"\nint main() {\n' + "".join(
        '  std::printf("%%u\\n", tsr::logprob_ctas(%dull, %dull, %s));\n' % (r, v, fits) for r, v in cases) + "}\n")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", os.path.join(ROOT, "tessera_b200", "csrc"),
                    str(tmp_path / "p.cpp"), "-o", str(tmp_path / "p")], check=True)
    got = subprocess.run([str(tmp_path / "p")], check=True, capture_output=True, text=True).stdout.split()
    for (rows, vocab), ctas in zip(cases, map(int, got)):
        sizes = [c for c in (2, 4, 8, 16) if rows * c <= (148 if c == 16 else 296) and vocab // c >= 1536]
        assert ctas == max([1] + [c for c in sizes if resident[c] > 0]), (rows, vocab)
