"""Instructions of whole warps (products, transposes, cluster barriers in their aligned form) are executed by converged warps.

Nothing converges a warp by itself behind a branch or a loop that goes by lane, or behind a wait, which lanes may leave one by one; where the
compiler joins them again is its own choice.  The sources are read statement by statement, loops twice, as a warp would run them.
"""
import re

import pytest

from sharq_b200._build import CSRC
from tests.test_dependent_launch_cpu import _code

ALIGNED = r"(?:movmatrix|ldmatrix4|ldmatrix4_trans|mma16816<\w+>|mma_f16|mma_f16_from0|cluster_sync)\s*\("
CONVERGES = r"__syncwarp\(\)|__syncthreads\(\)"
BY_LANE = r"\b(?:lane|g|t|chosen|threadIdx|col0|row|col)\b"
TOKEN = re.compile(rf"(?P<head>\b(?:if|for|while)\s*(?:constexpr\s*)?\()|(?P<sync>{CONVERGES})|(?P<aligned>{ALIGNED})"
                   rf"|(?P<apart>\bload\(\);|mbar_wait\()|(?P<open>\{{)|(?P<close>\}})|(?P<word>\belse\b)")


def _closing(text, at, pair):
    depth = 0
    for i in range(at, len(text)):
        depth += {pair[0]: 1, pair[1]: -1}.get(text[i], 0)
        if depth == 0:
            return i
    raise AssertionError("unbalanced")


def _statement_end(text, at):
    """Behind the statement that begins at `at`."""
    while text[at].isspace():
        at += 1
    if text[at] == "{":
        return _closing(text, at, "{}") + 1
    m = re.compile(r"(?:if|for|while)\s*(?:constexpr\s*)?\(").match(text, at)
    if m:
        at = _statement_end(text, _closing(text, m.end() - 1, "()") + 1)
        rest = re.compile(r"\s*else\b").match(text, at)
        return _statement_end(text, rest.end()) if rest else at
    depth = 0
    for i in range(at, len(text)):
        depth += {"(": 1, ")": -1, "{": 1, "}": -1}.get(text[i], 0)
        if text[i] == ";" and depth == 0:
            return i + 1
    raise AssertionError("no end")


def _run(text, at, end, converged, found):
    while True:
        m = TOKEN.search(text, at, end)
        if not m:
            return converged
        at = m.end()
        if m["sync"]:
            converged = True
        elif m["apart"]:
            converged = False
        elif m["aligned"]:
            if not converged:
                found.add(" ".join(text[max(0, m.start() - 60):m.end() + 20].split()))
        elif m["head"]:
            close = _closing(text, m.end() - 1, "()")
            condition, stop = text[m.end():close], _statement_end(text, close + 1)
            loop = not m["head"].startswith("if")
            by_lane = re.search(BY_LANE, condition)
            converged = _run(text, m.end(), close, converged, found)
            for _ in range(2 if loop else 1):
                converged = _run(text, close + 1, stop, converged and not by_lane, found)
            converged = converged and not by_lane
            at = stop


def unsound(text):
    """Places of whole-warp instructions behind lanes that have parted, in all kernels of a source text."""
    found = set()
    for m in re.finditer(r"__global__[^;{}]*?\b\w+_kernel\([^{}]*\)\s*\{", text):
        _run(text, m.end(), _closing(text, m.end() - 1, "{}"), True, found)
    return found


def test_what_the_reading_finds():
    """The reading itself, on small kernels."""
    body = "__global__ void some_kernel(int n) { %s }"
    good = ["if (n > 3) mma_f16(a); mma_f16(b);", "if (lane == 0) { x = 1; } __syncwarp(); mma_f16(b);",
            "for (int i = 0; i < n; ++i) { mma_f16(a); if (t < n) y = 1; __syncwarp(); }"]
    bad = ["if (lane == 0) x = 1; mma_f16(b);", "for (int i = 0; i < n; ++i) { mma_f16(a); if (t < n) y = 1; }",
           "if (t < n) mma_f16(a); __syncwarp();", "load(); ldmatrix4(a);", "for (int i = lane; i < n; i += 32) y = 1; movmatrix(a);",
           "while (n) { if (g < n) { y = 1; } cluster_sync(); }", "if (!mbar_wait(b)) x = 1; mma_f16(a);"]
    assert not any(unsound(body % b) for b in good)
    assert all(unsound(body % b) for b in bad)


@pytest.mark.parametrize("name", ["paged_attention.cu", "weight_only.cu"])
def test_kernels_of_the_decode_step(name):
    text = re.sub(r"^\s*#[^\n]*", "", _code(CSRC / name), flags=re.M)
    assert len(re.findall(ALIGNED, text)) > 3
    assert unsound(text) == set()


def test_a_result_used_by_some_lanes_is_made_by_all():
    """The transposes are volatile, so that they are not moved into the branch of the lanes that store them."""
    text = _code(CSRC / "paged_attention.cu")
    assert len(re.findall(r"movmatrix\.sync", text)) == len(re.findall(r"asm volatile\(\"movmatrix\.sync", text)) == 1
