"""CPU suite: a change of the build's flags reaches every object, in an incremental build too."""
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "streamingt2v_amd", "csrc")


def test_every_object_depends_on_the_makefile():
    """The flags that forbid packed fp32 instructions stand in the Makefile alone: objects built without them must not outlive a change."""
    base = subprocess.run(["make", "-C", CSRC, "-np", "all"], capture_output=True, text=True).stdout
    rules = dict(re.findall(r"^([\w/]+\.o): (.*)$", base, re.M))
    sources = {f[:-4] for f in os.listdir(CSRC) if f.endswith(".hip")}
    assert {o[:-2] for o in rules} >= sources
    for o in sources:
        assert "Makefile" in rules[o + ".o"].split(), o


def test_the_flags_forbid_packed_fp32():
    out = subprocess.run(["make", "-C", CSRC, "-nB", "all"], capture_output=True, text=True).stdout
    lines = [line for line in out.splitlines() if " -c " in line]
    assert lines and all("-Xclang -target-feature -Xclang -packed-fp32-ops" in line for line in lines)
