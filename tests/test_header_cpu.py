"""What the C header says of its version."""
from __future__ import annotations

import os
import re

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "gfa.h")


def test_the_version_is_described():
    """The number's comment begins with what that version brought."""
    number, first = re.search(r"#define GFA_VERSION (\d+) /\*\s*(\d+\.\d+\.\d+): \w+", open(HEADER).read()).groups()
    major, minor, patch = map(int, first.split("."))
    assert int(number) == 100 * major + 10 * minor + patch
