"""The Go bindings' calls that hand slices of the caller's length to the library: each checks it first (there is no Go toolchain here, so this reads
the source)."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def body(name):
    with open(os.path.join(ROOT, "go", "loomb200", "loomb200.go")) as f:
        text = f.read()
    found = re.search(r"^func \([^)]*\) %s\(.*?^}" % name, text, re.M | re.S)
    assert found, name
    return found.group(0)


def before(text, call, *checks):
    """Every check stands in front of the call."""
    at = text.index(call)
    for c in checks:
        assert -1 < text.find(c) < at, (call, c)


def test_sample_checks_its_slices():
    before(body("Sample"), "C.loom_b200_decoder_sample(", "C.loom_b200_decoder_batch(dec.d)", "len(params) != n", "logprobs != nil && len(logprobs) != n")
    text = body("Sample")
    assert text.index("len(params) != n") < text.index("&topK[0]")  # (an empty slice has no first entry)


def test_put_checks_its_slices():
    before(body("Put"), "C.loom_b200_adapters_put(", "C.loom_b200_adapters_info(", "len(down) != rank*int(cols)", "len(up) != rank*int(rows)")


def test_apply_takes_no_base():
    before(body("Apply"), "C.loom_b200_adapters_apply(", "if base != nil")
    assert len(re.findall(r"\bbase\.p\b", body("Apply"))) == 1
