"""Programmatic dependents read what the kernel before them may write by
plain loads. __ldg, and const __restrict__ pointers, which the compiler may
turn into it, are for memory that nobody writes while a kernel runs, and such
a kernel runs since before the wait for the one ahead of it: a scale, a row or
a length that the kernel ahead writes could be read stale. A race like that
shows on a GPU once in a long while, so the sources are read here."""
import glob
import os
import re

import pytest

from conftest import PKG

# weights and biases of the sampler, written when a handle is prepared
CONSTANT = {"kernels_fmt.cu": {"W", "b", "bx", "bc", "pos", "bmod", "bmod2", "bg4", "bs4", "bt4", "bv"},
            # (launched as a dependent by the sampler only)
            "kernels_gemm_tc.cu": {"p.bias"}}
FILES = sorted(os.path.basename(f) for f in glob.glob(os.path.join(PKG, "csrc", "*.cu"))
               if "pdl_wait()" in open(f).read())


def stale_loads(text, constant):
    """what a source reads as if it were constant, and is not"""
    names = re.findall(r"__ldg\(\s*\(?([\w.]+)", text)
    names += re.findall(r"const\s+\w+(?:\s+const)?\s*\*\s*__restrict__\s+(\w+)", text)
    names += re.findall(r"ld\.global\.nc\b", text)
    return sorted(set(names) - constant)


def test_files_are_found():
    assert {"kernels_attn.cu", "kernels_attn_tc.cu", "kernels_fmt.cu", "kernels_gemm_f8.cu", "kernels_gemm_tc.cu",
            "kernels_quant.cu"} <= set(FILES)


@pytest.mark.parametrize("name", FILES)
def test_dependents_read_by_plain_loads(name):
    with open(os.path.join(PKG, "csrc", name)) as f:
        assert stale_loads(f.read(), CONSTANT.get(name, set())) == []


def test_the_search_finds_them():
    text = "k(const float *__restrict__ a, const __half *b) { x = __ldg(p.q + 1) + __ldg(w[2] + i); }"
    assert stale_loads(text, {"w"}) == ["a", "p.q"]
