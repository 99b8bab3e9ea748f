"""The draw of a class asks for the row that its SM takes next: the one as many rows on as there are CTAs on the GPU at a time.  That is one an
SM as long as 1024 threads need more than half of its registers, read here from what the compiler said; results do not depend on it."""
import os
import re

import pytest

HERE = os.path.join(os.path.dirname(__file__), "..", "gpt.c_b200")


def test_the_row_that_comes_next():
    text = open(os.path.join(HERE, "csrc", "sample_sm100.cu")).read()
    assert "row + ahead < rows" in text
    distance = re.search(r"alone && C > 3 \? (.*) : 0\);", text).group(1)
    assert distance == "attn::sm_count()"


def test_one_cta_an_sm():
    log = os.path.join(HERE, "lib", "build.log")
    if not os.path.exists(log):
        pytest.skip("not built here")
    said = re.search(r"Compiling entry function '[^']*sample_kernelILi1024E.*?Used (\d+) registers", open(log).read(), re.S)
    assert int(said.group(1)) * 1024 * 2 > 65536
