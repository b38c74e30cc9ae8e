"""Kernels that may start before their predecessor ends: each waits for it on every path, as their sources show."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "chatlearn_b200", "csrc")


def _plain(text):
    """Source without comments."""
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def _kernels(path):
    """(name, body) of every kernel of a file."""
    text = _plain(open(path).read())
    for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\s*\((?:[^()]|\([^()]*\))*\)\s*)?(\w+)\s*\(", text):
        at = text.index("{", m.end())
        if ";" in text[m.end():at]:
            continue                                  # a declaration
        depth, end = 1, at + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield m.group(1), text[at:end]


ALL = {name: body for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))) for name, body in _kernels(path)}
EARLY = sorted(n for n, body in ALL.items() if "pdl_wait()" in body or "pdl_trigger()" in body)


def test_the_kernels_are_found():
    assert len(ALL) > 50
    assert {"paged_q8_kernel", "paged_q8_join_kernel", "q8_rows_kernel", "chunk_q8_kernel", "append_step_kernel", "append_pages_kernel",
            "token_logprob_kernel", "token_logprob_grad_kernel", "gemm_bf16_nt_kernel", "paged_decode_tc_kernel"} <= set(EARLY)


@pytest.mark.parametrize("name", EARLY)
def test_no_block_ends_before_it_has_waited(name):
    """A block that leaves before pdl_wait() lets its grid end early, and the next kernel with it."""
    body = ALL[name]
    assert "pdl_wait()" in body, "triggers its successor, but never waits for its predecessor"
    assert not re.search(r"\breturn\b", body[:body.index("pdl_wait()")])


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.cu"))), ids=os.path.basename)
def test_what_is_launched_early_waits(path):
    for name in re.findall(r"launch_pdl\(\s*(\w+)", _plain(open(path).read())):
        assert name in EARLY or name == "kernel", name
