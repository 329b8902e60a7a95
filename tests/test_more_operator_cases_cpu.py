"""The calls of perf/more_operators.py, without a GPU: every address they pass belongs to a
tensor that is alive when run() has returned, since the kernels run later."""
import ctypes

import pytest
import torch

from perf import more_operators as operators
from spar_amd import hip

CASES = [
    operators._append(3, 5, 4, 2, 16, 8, "interleaved", 5, 17, True),
    operators._attention(4, 2, 4, 2, 16, 1, 333, 0, 5, 2048, 0, 16),
    operators._attention(4, 2, 4, 2, 16, 3, 2048, 2048, 0, 50, 0, 5, "float64"),
    operators._beams(2, 3, 1000, 6, False, True, True, 7, 5, 9),
    operators._beams(1, 4, 300, 4, True, False, False, 1, 0, 0, "float64"),
]


def words(argument):
    """The 64-bit words of a call's argument, its structures' among them."""
    if isinstance(argument, int):
        return [argument]
    if isinstance(argument, (ctypes.Structure, ctypes.Array)):
        raw = bytes(argument)
        return [int.from_bytes(raw[i:i + 8], "little") for i in range(0, len(raw) - 7, 8)]
    return []


def tensors(value):
    if isinstance(value, torch.Tensor):
        yield value
    elif isinstance(value, dict):
        for x in value.values():
            yield from tensors(x)


@pytest.mark.parametrize("case", CASES, ids=lambda case: case["kind"])
def test_what_calls_write_outlives_them(monkeypatch, case):
    prepared, made = torch.device, torch.empty
    monkeypatch.setattr(operators.torch, "device", lambda name: prepared("cpu"))
    state = operators.prepare(case, 3)
    launched, spaces, passed, real = [], [], set(), hip.call

    def call(name, *arguments):
        if not name.startswith("spar_hip_launch"):
            return real(name, *arguments)  # host functions: workspace sizes
        launched.append(name)
        passed.update(word for argument in arguments for word in words(argument))

    def empty(*size, **options):
        tensor = made(*size, **options)
        spaces.append((tensor.data_ptr(), tensor.numel() * tensor.element_size()))
        return tensor

    monkeypatch.setattr(hip, "call", call)
    monkeypatch.setattr(operators.torch, "empty", empty)
    monkeypatch.setattr(operators, "own", True)
    made_by_run = operators.run(state)
    assert launched
    alive = [(x.untyped_storage().data_ptr(), x.untyped_storage().nbytes())
             for x in (*tensors(state), *tensors(made_by_run))]
    for address, size in spaces:
        if size and any(address <= word < address + size for word in passed):
            assert any(a <= address < a + n for a, n in alive), "a workspace that is freed"
    # a second pass writes the same workspaces, not new ones
    before = [x.data_ptr() for x in tensors(state.get("scratch", {}))]
    operators.run(state)
    assert before == [x.data_ptr() for x in tensors(state.get("scratch", {}))]
    assert bool(before) == (case["kind"] != "append")
