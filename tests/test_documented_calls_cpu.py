"""The C calls that the documents write out have the header's arguments, in its order.

Nearly all of them are untyped pointers: a call with two of them exchanged compiles."""
import pathlib
import re

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent
HEADER = re.sub(r"/\*.*?\*/", " ", (ROOT / "include" / "dash_attn.h").read_text(), flags=re.S)
PROTOTYPES = {name: [re.findall(r"\w+", a)[-1] for a in args.split(",")] for name, args in re.findall(r"\b(dash_\w+)\(([^()]*)\);", HEADER)}
# A document's shorter words for an argument.
WORDS = {"ws": "workspace", "ws_bytes": "workspace_bytes", "bytes": "positions_elem_bytes", "tables": "rope", "r": "rope", "k": "k_cache", "v": "v_cache"}


def arguments(text):
    """(function, its arguments as written) of every call in `text` that has any, whatever brackets are in them."""
    for m in re.finditer(r"\b(dash_\w+)\(", text):
        depth, at = 1, m.end()
        while depth and at < len(text):
            depth += {"(": 1, ")": -1}.get(text[at], 0)
            at += 1
        inside = re.sub(r"/\*.*?\*/", " ", text[m.end(): at - 1], flags=re.S)
        parts, depth = [""], 0
        for c in inside:
            depth += {"(": 1, ")": -1}.get(c, 0)
            if c == "," and depth == 0:
                parts.append("")
            else:
                parts[-1] += c
        if inside.strip():
            yield m.group(1), [p.strip() for p in parts]


# Calls whose arguments are plain names, the header's or WORDS' (a binding's own words, `query.ptr()` and the like, say nothing to a test).
CALLS = [(d.name, f, a) for d in [ROOT / "INTEGRATION.md", ROOT / "README.md"] for f, a in arguments(d.read_text())
         if f in PROTOTYPES and all(re.fullmatch(r"&?\w+", x) for x in a) and len(a) > 1]


@pytest.mark.parametrize("document,function,written", CALLS, ids=[c[1] for c in CALLS])
def test_a_documented_call_is_the_header_s(document, function, written):
    want = PROTOTYPES[function]
    names = [x.lstrip("&") for x in written]
    names = [x if x in want else WORDS.get(x, x) for x in names]
    assert len(names) == len(want), (document, written, want)
    assert names == want, (document, written, want)


def test_there_are_such_calls():
    assert any(f == "dash_rope_norm_apply" for _, f, _ in CALLS)
