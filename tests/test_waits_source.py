"""Every loop that waits inside a kernel ends by the clock (CPU, by reading the sources): whoever polls a barrier in shared memory or a counter
of other blocks does it with the shared waits, whose limit is a time, or compares the clock himself."""
import re

from jllm_serve_b200.csrc.build import CSRC

# what polls: a try on a barrier, a load of what another block counts up
POLLS = re.compile(r"mbarrier\.(?:try|test)_wait|mbar_try_wait\(|ld\.acquire\.gpu")


def loops(text):
    """The statements under every `while (...)` and `for (...)` of a source, with their heads."""
    for m in re.finditer(r"\b(?:while|for) \(", text):
        depth, i = 1, m.end()
        while depth:                                   # the head's closing parenthesis
            depth += {"(": 1, ")": -1}.get(text[i], 0)
            i += 1
        while text[i].isspace():
            i += 1
        if text[i] != "{":
            yield text[m.start():text.index(";", i) + 1]
            continue
        depth, j = 1, i + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[j], 0)
            j += 1
        yield text[m.start():j]


def test_loops_that_poll_look_at_the_clock():
    found = 0
    for path in sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")):
        for loop in loops(re.sub(r"//[^\n]*", "", path.read_text())):
            if POLLS.search(loop):
                found += 1
                assert "now_ns()" in loop, f"{path.name}: a loop that polls without a limit in time:\n{loop}"
    assert found >= 4


def test_no_wait_counts_tries_alone():
    for path in sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")):
        assert "SPIN_LIMIT" not in path.read_text(), path.name
