"""Wait states of hand-written loads to LDS, counted in the machine code that the build made.

gfx950 has the programmer (the compiler, outside of inline assembly) put at least

* one wait state between a write of m0 and a load to LDS, which takes its place in LDS from it;
* five between a vector instruction that writes a scalar register and a memory instruction that
  reads it, here a load's base or resource.

An instruction is a wait state, s_nop n is n + 1.  A load brings all of them with the write of its
m0, so that what the compiler puts in front does not matter."""

import re
import shutil
import subprocess
from pathlib import Path

import pytest

from gefen_amd import _lib

LLVM = Path("/opt/rocm/lib/llvm/bin")
OBJDUMP = str(LLVM / "llvm-objdump") if (LLVM / "llvm-objdump").exists() else shutil.which("llvm-objdump")
ADDRESS, M0 = 5, 1


@pytest.fixture(scope="module")
def listings(tmp_path_factory):
    """The instructions of each of the library's code objects; labels as None."""
    if OBJDUMP is None:
        pytest.skip("llvm-objdump is not installed")
    _lib.load()
    at = tmp_path_factory.mktemp("code")
    lib = shutil.copy(Path(_lib.__file__).resolve().parent / "libgefen_hip.so", at)
    subprocess.run([OBJDUMP, "--offloading", lib], cwd=at, check=True, stdout=subprocess.DEVNULL)
    objects = sorted(at.glob("*gfx950"))
    assert objects

    def read(path):
        out = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(path)], check=True,
                             capture_output=True, text=True).stdout
        lines = (line.split("//")[0].strip() for line in out.splitlines())
        return [None if line.endswith(">:") else line for line in lines if line.endswith(">:") or re.match("[a-z]+_", line)]

    return [read(p) for p in objects]


def states(line):
    op, _, rest = line.partition(" ")
    return int(rest.split()[0], 0) + 1 if op == "s_nop" else 1


def counted(listings, mnemonic):
    """For each load to LDS, the wait states between the last write of m0 and it, and those with
    that write."""
    for code in listings:
        for k, line in enumerate(code):
            if line is None or not line.startswith(mnemonic) or not re.search(r"_lds_|\blds\b", line):
                continue
            waited, at = 0, k - 1
            while code[at] is not None and not re.match(r"s_\w+ m0,", code[at]):
                waited += states(code[at])
                at -= 1
            assert code[at] is not None, "no write of m0 before " + line
            yield waited, waited + 1


def test_attention_waits_before_its_loads(listings):
    found = list(counted(listings, "global_load"))
    assert found
    assert min(m0 for m0, _ in found) >= M0
    assert min(base for _, base in found) >= ADDRESS


def test_linear_cross_entropy_waits_before_its_loads(listings):
    found = list(counted(listings, "buffer_load"))
    assert found
    assert min(m0 for m0, _ in found) >= M0
    assert min(base for _, base in found) >= ADDRESS
