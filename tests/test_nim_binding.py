"""What can be checked of the Nim host layer without a Nim compiler: that nothing it declares is called by a word that Nim
keeps for itself. The parser stops there, and takes every binding of the file with it."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FILES = ("hip_abi.nim", "tensor_hip.nim")
# The keywords of the Nim manual ("Lexical Analysis", identifiers and keywords).
KEYWORDS = set("""addr and as asm bind block break case cast concept const continue converter defer discard distinct div do elif
else end enum except export finally for from func if import in include interface is isnot iterator let macro method mixin mod
nil not notin object of or out proc ptr raise ref return shl shr static template try tuple type using var when while xor
yield""".split())


def normal(name):
    """Nim's comparison of names: the first letter counts as it stands, the others without case and underscores."""
    return name[:1] + name[1:].replace("_", "").lower()


def uncommented(text):
    text = re.sub(r'"(?:[^"\\\n]|\\.)*"', '""', text)
    return re.sub(r"#[^\n]*", "", text)


def declared(text):
    """Names of procs and templates and of their parameters, of constants, variables, tuple fields and types; not quoted ones."""
    text = uncommented(text)
    names = re.findall(r"\b(?:proc|template|func|iterator|macro|converter)\s+(\w+)", text)
    names += re.findall(r"\b(?:let|var|const|for)\s+(\w+)", text)
    for group in re.findall(r"\b(?:let|var)\s+\(([^)]*)\)", text) + re.findall(r"\bfor\s+([\w, ]+)\bin\b", text):
        names += re.findall(r"\w+", group)
    # `a, b: T` in parameter lists, tuples, objects and declaration blocks, and `NAME* = value`
    for group in re.findall(r"((?:\w+\*?\s*,\s*)*\w+\*?)\s*:\s*(?=[A-Za-z_\[])", text):
        names += re.findall(r"\w+", group)
    names += re.findall(r"^\s+(\w+)\*?\s*=\s", text, flags=re.M)
    return names


@pytest.mark.parametrize("name", FILES)
def test_nothing_is_called_by_a_keyword(name):
    with open(os.path.join(ROOT, "nim", name)) as f:
        names = declared(f.read())
    assert len(names) > 100
    words = {normal(k) for k in KEYWORDS}
    # `else:` and `try:` and the like end in the colon that a declaration has too
    blocks = {normal(k) for k in ("else", "try", "finally", "except", "block", "static", "defer", "do")}
    bad = sorted({n for n in names if normal(n) in words - blocks})
    assert not bad, f"nim/{name} declares {bad}"


def test_the_check_sees_parameters_variables_and_fields():
    seen = declared("proc f*(a, out: ptr cfloat; b: int): tuple[x, end: int] = discard\nlet (of, c) = g()\nconst\n  mod* = 1\n# var is: int\n")
    assert {"f", "a", "out", "b", "x", "end", "of", "c", "mod"} <= set(seen) and "is" not in seen


def body(name):
    """The text of one proc of nim/tensor_hip.nim."""
    with open(os.path.join(ROOT, "nim", "tensor_hip.nim")) as f:
        text = f.read()
    found = re.search(rf"^proc {name}\*?\[.*?(?=^(?:proc|template|type|#) ?)", text, flags=re.M | re.S)
    assert found, name
    return found.group(0)


def test_the_statistics_of_group_norm_are_looked_at_before_they_are_read():
    """mean, rstd and the gradient go to the device as bare pointers: their shapes and their order in memory are checked first."""
    calls = body("group_norm_backward")
    check = calls.index("checkNormGradients(grad_output, x, mean, rstd, groups)")
    assert check < calls.index("mean.get_offset_ptr") and check < calls.index("newHipTensor")
    checks = body("checkNormGradients")
    for what in ("grad_output.shape != x.shape", "mean.rank != 2", "mean.shape[0] != x.shape[0]", "mean.shape[1] != groups", "rstd.shape != mean.shape"):
        assert what in checks
    for t in ("grad_output", "mean", "rstd"):
        assert f"not {t}.is_C_contiguous" in checks


@pytest.mark.parametrize("name", ["decay_attention", "decay_attention_backward"])
def test_padded_batches_reach_the_device(name):
    text = body(name)
    assert "lengths = default(HipTensor[int64])" in text and "checkLengths(lengths" in text and "log_decay.get_offset_ptr, lengths.ptrOrNil" in text


@pytest.mark.parametrize("name,optional", [("rotate", ["positions"]), ("decay_attention", ["first", "lengths"]), ("decay_attention_backward", ["state", "grad_state", "lengths"]),
                                           ("group_norm", ["weight", "bias"]), ("group_norm_backward", ["weight", "bias"])])
def test_what_may_be_left_out_is_handed_on_as_nil(name, optional):
    text = body(name)
    for t in optional:
        assert f" {t}.ptrOrNil" in text and not re.search(rf"\b{t}\.get_offset_ptr", text)
