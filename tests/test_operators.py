"""perf/operators.py: before it makes any input, the program's torch work is on
the context's stream, which waits for no other."""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Stop(Exception):
    pass


@pytest.mark.parametrize("own", [True, False])
def test_inputs_are_made_on_the_calls_stream(monkeypatch, own):
    spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = own
    did = []

    class Stream:
        def wait_stream(self, other):
            did.append(("wait", other))

    mine = Stream()

    def generator(**kw):
        did.append("inputs")
        raise Stop

    monkeypatch.setattr(m, "_context", lambda: (None, mine))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: "default")
    monkeypatch.setattr(torch.cuda, "set_stream", lambda s: did.append(("set", s)))
    monkeypatch.setattr(torch, "Generator", generator)
    for case in m.listed():
        did.clear()
        with pytest.raises(Stop):
            m.prepare(case, 1)
        assert did == ([("wait", "default"), ("set", mine)] if own else []) + ["inputs"], case["name"]
