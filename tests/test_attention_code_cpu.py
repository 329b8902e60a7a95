"""The attention kernels' source and their code in the built library, without a GPU."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from spar_amd import hip

SOURCES = Path(__file__).resolve().parent.parent / "spar_amd" / "csrc" / "hip"
OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")


def statements(text):
    """The asm statements of a source, from `asm` to the semicolon behind."""
    return re.findall(r"\basm(?:\s+volatile)?\s*\(.*?\)\s*;", text, re.S)


def test_asm_names_the_registers_it_writes():
    """An instruction that writes m0 inside asm is unknown to the compiler, which may keep
    a value of its own there, unless the statement names it among what it changes."""
    seen = 0
    for path in sorted([*SOURCES.glob("*.hip"), *SOURCES.glob("*.hpp")]):
        for statement in statements(path.read_text()):
            if re.search(r"\bm0\s*,", statement):
                seen += 1
                assert statement.rsplit(":", 1)[1].count('"m0"') == 1, (path.name, statement)
    assert seen >= 1


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """Instructions of the library's attention kernels, by name."""
    if not OBJDUMP.exists():
        pytest.skip("no llvm-objdump")
    folder = tmp_path_factory.mktemp("code")
    library = folder / "library.so"
    shutil.copy(hip.library_path(), library)
    subprocess.run([OBJDUMP, "--offloading", library], cwd=folder, check=True,
                   capture_output=True, timeout=120)
    found = {}
    for code in sorted(folder.glob("*gfx950*")):
        if b"9attention" not in code.read_bytes():  # the namespace in the symbols' names
            continue
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", code], check=True,
                              capture_output=True, text=True, timeout=300).stdout
        name = None
        for line in text.splitlines():
            label = re.match(r"[0-9a-f]+ <(.*)>:", line)
            if label:
                name = label[1]
                found[name] = []
                continue
            instruction = line.split("//")[0].strip()
            if name is not None and instruction:
                found[name].append(instruction)
    return {name: code for name, code in found.items() if "attention" in name}


def test_no_masked_block_is_empty(kernels):
    """A short-circuited condition that selects between a matrix product's result and a
    constant has been compiled to a block that saves and restores the mask of lanes around
    nothing: the selected value was always the constant.  None of the kernels has one."""
    assert any("tile_kernel" in name for name in kernels)
    assert any("key_kernel" in name for name in kernels)
    for name, code in kernels.items():
        for first, second in zip(code, code[1:]):
            saves = re.match(r"s_(and|or|andn2)_saveexec_b64|s_and_b64 exec", first)
            assert not (saves and re.match(r"s_(or|mov)_b64 exec", second)), (name, first, second)


def test_m0_is_written_by_the_loads_to_lds_alone(kernels):
    for name, code in kernels.items():
        for i, instruction in enumerate(code):
            if re.search(r"\bm0\b", instruction):
                assert instruction.startswith("s_mov_b32 m0, s"), (name, instruction)
                assert code[i + 1] == "s_nop 0", (name, code[i:i + 3])
                assert code[i + 2].startswith("global_load_lds_dwordx4"), (name, code[i:i + 3])
