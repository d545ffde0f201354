"""Every C name that INTEGRATION.md gives is declared by a header under include/, so that a caller who follows it can link."""
from __future__ import annotations

import re
from pathlib import Path

from test_abi import HEADERS, declared_functions

TEXT = (Path(__file__).resolve().parent.parent / "INTEGRATION.md").read_text()


def test_named_functions_are_declared():
    named = set(re.findall(r"\b(dsv4_[a-z0-9_]+)\(", TEXT))
    assert len(named) > 15 and named <= {f for _, f in declared_functions()}


def test_named_words_are_in_a_header():
    words = {w for w in re.findall(r"\b(dsv4_[a-z0-9_]+[a-z0-9])\b(?!\.)", TEXT) if f"lib{w}" not in TEXT}
    headers = "".join(h.read_text() for h in HEADERS)
    assert not {w for w in words if w not in headers}
