"""Every script that builds the library takes its units and flags from csrc/flags.sh."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "instant-nsr-pl_amd", "csrc")
SCRIPTS = [os.path.join(CSRC, "build.sh"), os.path.join(ROOT, "tools", "build_variants.sh"),
           os.path.join(ROOT, "tools", "build_baseline.sh")]


def _flags(expression):
    return subprocess.check_output(["bash", "-c", f'. "{CSRC}/flags.sh"; echo {expression}'], text=True).split()


def test_units_are_all_sources():
    units = _flags("$NSR_UNITS")
    assert sorted(units) == sorted(f[:-4] for f in os.listdir(CSRC) if f.endswith(".hip"))
    assert _flags("$(nsr_objects /o)") == [f"/o/{u}.o" for u in units]
    assert _flags("$(nsr_objects /o hashgrid)") == [f"/o/{u}.o" for u in units if u != "hashgrid"]


def test_scripts_have_no_units_or_flags_of_their_own():
    assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in " ".join(_flags("$NSR_FLAGS"))
    for path in SCRIPTS:
        text = open(path).read()
        assert re.search(r'^\. "\$\w+/flags\.sh"$', text, re.M), path
        compiles = [line for line in text.splitlines() if re.search(r"\bhipcc\b.* -c ", line)]
        assert compiles and all("hipcc $NSR_FLAGS " in line for line in compiles), path
        assert "$(nsr_objects " in text and "-ffp-contract" not in text and "occupancy" not in text, path
        subprocess.check_call(["bash", "-n", path])


def test_single_file_tools_are_compiled_alike():
    """the compile lines in the headers of tools/*.hip leave packed fp32 instructions out too"""
    for name in os.listdir(os.path.join(ROOT, "tools")):
        if name.endswith(".hip"):
            for line in open(os.path.join(ROOT, "tools", name)):
                if "hipcc --offload-arch" in line:
                    assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in line, name
