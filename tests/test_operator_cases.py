"""perf/operators.py on the CPU: the framework's calls of a pass, with a library that notes them."""
import ctypes
import importlib.util
import os
from types import SimpleNamespace

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Notes:
    """Stands for the bindings and the library: every call is noted with its last argument, the stream."""

    def __init__(self):
        self.calls = []

    def lib(self):
        return self

    def check(self, rc):
        assert rc == 0

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a[-1])) or 0


@pytest.mark.parametrize("case,names", [({"kind": "append", "cache": "f16"}, ["af_kv_append"]),
                                        ({"kind": "append", "cache": "q4"}, ["af_kv_append", "af_kv_read"]),
                                        ({"kind": "attend"}, ["af_paged_attention"]), ({"kind": "select"}, ["af_logits_select"])], ids=str)
def test_a_pass_runs_on_the_stream_current_at_its_call(monkeypatch, case, names):
    spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
    cases = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(cases)
    cases.own = True
    # ctypes structs of arrays that no call here reads
    inner = type("Inner", (ctypes.Structure,), {"_fields_": [("x", ctypes.c_uint32)]})
    args = type("Args", (ctypes.Structure,), {"_fields_": [("pages", inner), ("batch", inner)]})()
    t = torch.zeros(1)
    notes = Notes()
    state = {"case": case, "native": notes, "device": 0, "args": args, "values": [t, t],
             **{n: t for n in ("q", "k", "v", "q_out", "out", "k_pages", "v_pages", "result")}}
    for stream in (11, 12):
        monkeypatch.setattr(torch.cuda, "current_stream", lambda *_, s=stream: SimpleNamespace(cuda_stream=s))
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda _, s=stream: s, raising=False)
        notes.calls.clear()
        cases.run(state)
        assert notes.calls == [(n, stream) for n in names]
