"""perf/operators.py lends torch's memory to the library and back: torch works on the library's stream before the first call that does
so, after everything that torch had queued elsewhere. Checked with recorders in the place of the streams and of the library."""
import importlib.util
import os
import sys
import types

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
torch = pytest.importorskip("torch")


def test_torch_joins_the_librarys_stream_before_the_first_call(monkeypatch):
    spec = importlib.util.spec_from_file_location("sequence_cases", os.path.join(ROOT, "perf", "operators.py"))
    cases = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(cases)
    done = []

    class Stream:
        def __init__(self, pointer):
            done.append(("stream", pointer))

        def wait_stream(self, other):
            done.append(("waits for", other))

    library = types.SimpleNamespace(am_hip_stream=lambda: 0x5)
    am = types.SimpleNamespace(sync=lambda: done.append("sync"), load_library=lambda: library, HipTensor=lambda *a: "tensor", Layout=lambda *a: None,
                               group_norm=lambda *a, **k: done.append("call"))
    monkeypatch.setitem(sys.modules, "arraymancer_amd", am)
    monkeypatch.setattr(torch.cuda, "ExternalStream", Stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: "torch's")
    monkeypatch.setattr(torch.cuda, "set_stream", lambda s: done.append(("torch on", type(s))))
    monkeypatch.setattr(cases, "own", True)
    state = dict(case=dict(kind="norm", train=False, groups=2, activation="none"), x=torch.zeros(2, 4), weight=None, bias=None)
    cases.run(state)
    cases.run(state)
    assert done == ["sync", ("stream", 0x5), ("waits for", "torch's"), ("torch on", Stream), "call", "call"]
