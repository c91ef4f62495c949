"""Kernels that start before the one ahead of them has finished
(griddepcontrol.wait): what that one writes must not be declared constant for
the kernel's lifetime.  `const T *__restrict__` admits the read-only load path,
which is not coherent with a kernel still writing, and such loads may be moved
above the wait."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "chelis_b200", "csrc")
# arguments that were complete before the kernel ahead began
COMPLETE = {"sort_place_kernel": {"ids"}}


def _kernels():
    """(name, parameters, body) of every kernel."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        with open(path) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for m in re.finditer(r"__global__\s+void\s+[^;{]*?(\w+_kernel)\s*\(", text):
            depth, i = 1, m.end()
            while depth:
                depth += {"(": 1, ")": -1}.get(text[i], 0)
                i += 1
            start = body = text.index("{", i)
            depth = 0
            while True:
                depth += {"{": 1, "}": -1}.get(text[body], 0)
                body += 1
                if depth == 0:
                    break
            yield m.group(1), text[m.end():i - 1], text[start:body]


def test_no_wait_outside_the_kernels_found():
    waits = 0
    for path in glob.glob(os.path.join(CSRC, "*.cu*")):
        with open(path) as f:
            waits += re.sub(r"//[^\n]*", "", f.read()).count("griddepcontrol.wait")
    assert waits == sum(body.count("griddepcontrol.wait") for _, _, body in _kernels()) > 0


def test_dependent_kernels_declare_nothing_constant_that_is_still_written():
    seen = set()
    for name, params, body in _kernels():
        if "griddepcontrol.wait" not in body:
            continue
        seen.add(name)
        constant = {m.group(1) for m in re.finditer(r"const\s+[\w:]+\s*\*\s*__restrict__\s+(\w+)", params)}
        assert constant <= COMPLETE.get(name, set()), f"{name}: {constant}"
        assert "__ldg" not in body, name
    assert {"sort_scan_kernel", "sort_place_kernel", "scaled8_kernel"} <= seen
