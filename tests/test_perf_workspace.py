"""The performance cases' workspace (perf/operators.py), with a stand-in for torch: calls
on two streams may overlap and must not share one."""
import importlib.util
import sys
import types
from pathlib import Path

CASES = Path(__file__).resolve().parent.parent / "perf" / "operators.py"


class _Tensor:
    count = 0

    def __init__(self, n, **_):
        _Tensor.count += 1
        self.n, self.ptr = n, 4096 * _Tensor.count

    def numel(self):
        return self.n

    def data_ptr(self):
        return self.ptr


def test_each_stream_has_its_own_workspace(monkeypatch):
    torch = types.ModuleType("torch")
    current = types.SimpleNamespace(device_index=0, cuda_stream=1, device="cuda:0")
    torch.cuda = types.SimpleNamespace(current_stream=lambda: current)
    torch.uint8, torch.empty = "uint8", _Tensor
    monkeypatch.setitem(sys.modules, "torch", torch)
    spec = importlib.util.spec_from_file_location("perf_operators_under_test", CASES)
    cases = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(cases)
    seen = set()
    for current.device_index, current.cuda_stream in ((0, 1), (0, 2), (1, 1)):
        at = cases._workspace(1000)
        assert at not in seen
        seen.add(at)
        assert cases._workspace(500) == at                   # kept while it is large enough
    current.device_index, current.cuda_stream = 0, 2
    larger = cases._workspace(2000)
    assert larger not in seen and cases._workspace(2000) == larger
