"""perf/operators.py on the CPU: preparing a case makes its inputs and nothing
else (no handle, no layout of weights), the same whichever side runs them."""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture()
def ops(monkeypatch):
    spec = importlib.util.spec_from_file_location("operator_cases", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    monkeypatch.setattr(m, "DEV", "cpu")
    return m


CASES = [
    dict(op="verify", B=3, K=2, V=90, dtype="f32", draft="rows", ragged=True, mask=True, cut=True, greedy=True, pad=3),
    dict(op="tree", B=2, branch="2.1", V=70, dtype="bf16", draft="given", ragged=False, greedy=False, pad=0),
    dict(op="head", B=2, H=128, V=300, group=64, out="f32"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: c["op"])
def test_inputs_are_all_that_is_prepared(ops, monkeypatch, case):
    plain = ops.prepare(case, 5)

    def used():
        raise AssertionError("the package is not needed to prepare inputs")

    monkeypatch.setattr(ops, "_package", used)
    monkeypatch.setattr(ops, "own", True)
    s = ops.prepare(case, 5)
    assert s.keys() == plain.keys()
    for k, v in s.items():
        if isinstance(v, torch.Tensor):
            assert torch.equal(v, plain[k]), k
        else:
            assert v == plain[k], k


def test_one_handle_serves_every_call(ops, monkeypatch):
    made = []

    class Package:
        @staticmethod
        def Sampler(device, **limits):
            made.append(device)
            return object()

    device = [0]
    monkeypatch.setattr(torch.cuda, "current_device", lambda: device[0])
    a, b = ops._handle(Package), ops._handle(Package)
    assert a is b and made == [0]
    device[0] = 1
    assert ops._handle(Package) is not a and made == [0, 1]
