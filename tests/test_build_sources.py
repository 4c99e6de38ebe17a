"""What the build files say about the sources.  No GPU is needed."""
import os
import re

PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fp6_llm_amd")


def included(path):
    """Every file of this tree that a source includes, itself or through another."""
    found = set()
    with open(path) as f:
        names = re.findall(r'^\s*#include "([^"]+)"', f.read(), re.M)
    for name in names:
        at = os.path.normpath(os.path.join(os.path.dirname(path), name))
        if os.path.exists(at):
            found |= {at} | included(at)
    return found


def test_objects_of_the_makefile_depend_on_all_that_they_include():
    with open(os.path.join(PACKAGE, "Makefile")) as f:
        text = f.read()
    headers = re.search(r"^HDRS = (.*)$", text, re.M).group(1)
    rules = re.findall(r"^\$\(OBJ\)/(\S+)\.o: (.*)$", text, re.M)
    assert len(rules) == 5
    for target, needs in rules:
        needs = [os.path.normpath(os.path.join(PACKAGE, n)) for n in needs.replace("$(HDRS)", headers).split()]
        missing = included(needs[0]) - set(needs)
        assert not missing, "%s.o: %s" % (target, sorted(os.path.basename(m) for m in missing))


def test_internal_functions_have_callers():
    csrc = os.path.join(PACKAGE, "csrc")
    with open(os.path.join(csrc, "fp6mi_internal.h")) as f:
        header = re.sub(r"//.*", "", f.read())
    declared = re.findall(r"^(?:int|size_t|void|LaunchCfg)\s+(\w+)\(", header, re.M)
    assert {"run_linear", "linear_shape", "prepack_ref"} <= set(declared)
    text = ""
    for name in sorted(os.listdir(csrc)):
        if name.endswith((".hip", ".cpp", ".inc")):
            with open(os.path.join(csrc, name)) as f:
                text += re.sub(r"//.*", "", f.read())
    for name in declared:   # (the definition, and a call at least)
        assert len(re.findall(r"\b%s\(" % name, text)) >= 2, name
