"""Warps that meet on a named barrier have to reach it whatever became of their bounded waits: one that leaves early would keep the
others standing there.  So no loop around such a barrier may be left by `break` or `return`, or end on a wait's result."""
import glob
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BARRIER = re.compile(r'"bar\.(?:sync|arrive) \d|\bnamed_(?:sync|arrive)\(group')


def source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(ROOT, "apnn_tc_b200", "csrc", name)).read())


def closing(text, at):
    """Behind the brace or parenthesis that closes the one at `at`."""
    opens, closes = text[at], {"(": ")", "{": "}"}[text[at]]
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == opens) - (text[i] == closes)
        if depth == 0:
            return i + 1
    raise AssertionError("unbalanced")


def loops_around_barriers(text):
    """(header, body) of every `for` whose body holds a named barrier."""
    for m in re.finditer(r"\bfor \(", text):
        head = closing(text, m.end() - 1)
        start = head + len(text[head:]) - len(text[head:].lstrip())
        end = closing(text, start) if text[start] == "{" else text.index(";", start)
        if text[start:].startswith("for ("):      # a loop over a loop, without braces
            inner = closing(text, text.index("(", start))
            end = closing(text, text.index("{", inner))
        if BARRIER.search(text[start:end]):
            yield text[m.end():head - 1], text[start:end]


@pytest.mark.parametrize("name,least", [("kv4_prompt.cu", 1), ("linear_tile.cu", 5)])
def test_no_wait_keeps_a_warp_from_a_named_barrier(name, least):
    assert os.path.join(ROOT, "apnn_tc_b200", "csrc", name) in glob.glob(os.path.join(ROOT, "apnn_tc_b200", "csrc", "*.cu"))
    seen = 0
    for head, body in loops_around_barriers(source(name)):
        seen += 1
        assert not re.search(r"\b(break|return|goto)\b", body), f"{name}: for ({head}) is left early"
        assert not re.search(r"\bok\b", head), f"{name}: for ({head}) ends on a wait's result"
    assert seen >= least
