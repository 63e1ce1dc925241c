"""Loads and stores through buffer descriptors: the descriptor's end is checked against the vector offset (with the
immediate one) alone, so no kernel puts a part of an address into the scalar offset."""
from __future__ import annotations

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "fastmoe_amd" / "csrc"
CALL = re.compile(r"__builtin_amdgcn_raw_(?:ptr_)?buffer_(load|store)(_lds)?\w*\(")


def arguments(text, start):
    """The arguments of the call whose opening parenthesis ends at `start`."""
    out, depth, at = [], 0, start
    for i in range(start, len(text)):
        if text[i] in "([{":
            depth += 1
        elif text[i] in ")]}":
            if depth == 0:
                return out + [text[at:i].strip()]
            depth -= 1
        elif text[i] == "," and depth == 0:
            out.append(text[at:i].strip())
            at = i + 1
    raise AssertionError("a call without an end")


def test_no_access_has_a_scalar_offset():
    seen = 0
    for path in sorted(CSRC.iterdir()):
        if path.suffix not in (".hip", ".h"):
            continue
        text = path.read_text()
        for m in CALL.finditer(text):
            args = arguments(text, m.end())
            # load(descriptor, vector, scalar, policy), store(value first), load_lds(descriptor, to, size, vector, scalar, ...)
            scalar = args[4 if m.group(2) else 2 if m.group(1) == "load" else 3]
            assert scalar == "0", (path.name, text.count("\n", 0, m.start()) + 1, scalar)
            seen += 1
    assert seen >= 10  # the pattern finds them
