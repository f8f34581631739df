"""The tables of the repository's documents: every row has its heading's cells."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _cells(line):
    line = re.sub(r"`[^`]*`", "code", line.strip()).replace("\\|", "bar")  # a bar inside code or behind a backslash is text
    return line.count("|") - 1 if line.endswith("|") else -1


@pytest.mark.parametrize("name", ["README.md", "DESIGN.md", "INTEGRATION.md"])
def test_rows_have_their_headings_cells(name):
    want, wrong = 0, []
    for number, line in enumerate(open(os.path.join(ROOT, name), encoding="utf-8"), 1):
        if not line.startswith("|"):
            want = 0
            continue
        want = want or _cells(line)
        if _cells(line) != want:
            wrong.append(f"{number}: {line[:60]}")
    assert not wrong, wrong
