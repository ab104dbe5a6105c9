"""The operators of a decoder through the C++ host layer, alone
and as a run (tests/cpp/decoder_tests.cpp). The binary runs once; each case is
reported as its own pytest item."""
import os
import re
import subprocess

import pytest

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
BIN = os.path.join(HERE, "cpp", "decoder_tests")


def case_names():
    text = open(BIN + ".cpp").read()
    return re.findall(r'\{"(\w+)",', text[text.index("const Case kCases[]"):])


@pytest.fixture(scope="module")
def results():
    if not os.path.exists(BIN):
        pytest.fail(f"test binary missing: {BIN} (run __graft_entry__.build())")
    print(f"running {BIN}", flush=True)
    proc = subprocess.run([BIN], capture_output=True, text=True, timeout=100)
    found = re.findall(r"^(PASS|FAIL) (\w+)(?:: (.*))?$", proc.stdout, re.M)
    return {name: (status, why) for status, name, why in found}, proc.stdout[-1500:] + proc.stderr[-1500:]


@pytest.mark.parametrize("name", case_names())
def test_case(results, name):
    found, tail = results
    assert name in found, f"{name} did not report:\n{tail}"
    assert found[name][0] == "PASS", found[name][1]
