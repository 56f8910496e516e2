"""build() of __graft_entry__.py: the library comes first, and the test programs beside it are made only where the Makefile of
tests/cpp knows them."""
import os
import re
import shutil

import pytest

import __graft_entry__ as entry
import am_oracle
import arraymancer_amd
from arraymancer_amd import build as hip_build

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")


@pytest.fixture
def steps(monkeypatch):
    """What build() does, in order, without doing it."""
    done = []
    monkeypatch.setattr(hip_build, "build", lambda **kw: done.append("library"))
    monkeypatch.setattr(arraymancer_amd, "load_library", lambda: done.append("load"))
    monkeypatch.setattr(am_oracle, "build", lambda **kw: done.append("oracle"))
    monkeypatch.setattr("subprocess.run", lambda cmd, **kw: done.append(cmd))
    return done


def test_the_library_is_built_and_loaded_before_the_test_programs(steps):
    entry.build()
    assert steps[:2] == ["library", "load"] and steps[2] == "oracle" and len(steps) == 4
    assert steps[3][0] == "make" and {"test_tensor_hip", "test_tensor_hip_asan", "test_display_host"} <= set(steps[3])


@pytest.mark.parametrize("missing", ["rule", "source", "makefile"])
def test_a_program_that_the_makefile_does_not_know_is_left_out(tmp_path, missing, steps, monkeypatch):
    for name in os.listdir(CPP):
        if name.endswith(".cpp") or name == "Makefile":
            shutil.copy(os.path.join(CPP, name), tmp_path / name)
    make = tmp_path / "Makefile"
    if missing == "rule":
        make.write_text(re.sub(r"^test_sequence:.*?(?=^\S|^$)", "", make.read_text(), flags=re.M | re.S))
    elif missing == "source":
        os.remove(tmp_path / "test_sequence.cpp")
    else:
        os.remove(make)
    got = entry.cpp_programs(str(tmp_path))
    assert got == ([] if missing == "makefile" else [p for p in entry.CPP_PROGRAMS if p != "test_sequence"])
    monkeypatch.setattr(entry, "CPP_TESTS", str(tmp_path))
    monkeypatch.setattr(entry, "cpp_programs", lambda: got)
    entry.build()
    assert steps[:3] == ["library", "load", "oracle"] and not any("test_sequence" in s for s in steps)
