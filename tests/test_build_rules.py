"""The Makefile's rule names every header that a source includes, directly or through another: an edit recompiles what depends on it."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tensorcore_b200", "csrc")


def _included(name, seen):
    path = os.path.normpath(os.path.join(CSRC, name))
    if path in seen or not os.path.exists(path):
        return seen
    seen.add(path)
    for other in re.findall(r'^\s*#include "([^"]+)"', open(path).read(), re.M):
        for base in (os.path.dirname(path), os.path.join(CSRC, "..", "..", "include")):
            if os.path.exists(os.path.join(base, other)):
                _included(os.path.join(base, other), seen)
                break
    return seen


def test_headers_are_prerequisites():
    rules = dict(re.findall(r"^\$\(OBJ\)/%\.o: %(\.\w+) (.*)$", open(os.path.join(CSRC, "Makefile")).read(), re.M))
    assert sorted(rules) == [".cpp", ".cu"]
    for suffix, named in rules.items():
        named = {os.path.normpath(os.path.join(CSRC, f)) for f in named.split()}
        for source in sorted(f for f in os.listdir(CSRC) if f.endswith(suffix)):
            missing = _included(source, set()) - named - {os.path.join(CSRC, source)}
            assert not missing, (source, sorted(os.path.basename(m) for m in missing))
