"""The workspace of the second set of performance cases (perf/more_operators.py), with a stand-in
for torch: calls on two streams may overlap and must not share one."""
import test_perf_workspace as first


def test_each_stream_has_its_own_workspace(monkeypatch):
    monkeypatch.setattr(first, "CASES", first.CASES.with_name("more_operators.py"))
    first.test_each_stream_has_its_own_workspace(monkeypatch)
