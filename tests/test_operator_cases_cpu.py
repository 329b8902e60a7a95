"""The calls of perf/operators.py, without a GPU: every address they pass belongs to a
tensor that is alive when run() has returned, since the kernels run later."""
import ctypes

import pytest
import torch

from perf import operators
from spar_amd import hip

CASES = [
    operators._rotary(2, 3, 2, 8, 8, "half", 5, "none", True),
    operators._norm(2, 3, 4, 2, 8, 4, "interleaved", 5, "parts", True),
    operators._attention(2, 4, 2, 16, 40, 40, 30, 8, 2, False, True),
    operators._attention(2, 4, 2, 16, 1, 4096, 3000, 0, 0, True, False),
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
    assert bool(before) == (case["kind"] != "rotary")
