"""Copies from memory to LDS in the built library's device code: the LDS address in M0 has to be written a wait state before
the copy that reads it.  No device call is made; what is read is the code that was built here."""

import os
import shutil
import struct
import subprocess
import tempfile
from concurrent.futures import ThreadPoolExecutor

import pytest

from boundflow_amd import _lib
from boundflow_amd.build import ARCH, hipcc

BUNDLE = b"__CLANG_OFFLOAD_BUNDLE__"


def device_code():
    """The device objects of the library: a bundle a translation unit, its entries (offset, size, target)."""
    data = _lib.LIB_PATH.read_bytes()
    at = data.find(BUNDLE)
    while at >= 0:
        entry = at + len(BUNDLE) + 8
        for _ in range(struct.unpack_from("<Q", data, entry - 8)[0]):
            offset, size, length = struct.unpack_from("<QQQ", data, entry)
            if ARCH.encode() in data[entry + 24:entry + 24 + length] and size:
                yield data[at + offset:at + offset + size]
            entry += 24 + length
        at = data.find(BUNDLE, at + 1)


def test_m0_is_written_a_wait_state_before_a_copy_reads_it():
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built (run python -m boundflow_amd.build)")
    objdump = shutil.which("llvm-objdump") or os.path.join(
        os.path.dirname(os.path.dirname(os.path.realpath(hipcc()))), "lib", "llvm", "bin", "llvm-objdump")
    if not os.path.exists(objdump):
        pytest.skip("no llvm-objdump")

    def copies(code):
        """(copies, those right behind a write of M0)"""
        with tempfile.NamedTemporaryFile(suffix=".co") as f:
            f.write(code)
            f.flush()
            text = subprocess.run([objdump, "-d", "--no-show-raw-insn", "--no-leading-addr", f.name], capture_output=True,
                                  text=True, check=True).stdout
        seen, late, last = 0, 0, []
        for words in (line.replace(",", " ").split() for line in text.splitlines()):
            if words and "load_lds" in words[0]:
                seen += 1
                late += last[:1] != [] and last[0].startswith("s_") and last[1:2] == ["m0"]
            last = words or last
        return seen, late

    with ThreadPoolExecutor(8) as pool:
        counts = list(pool.map(copies, device_code()))
    assert sum(seen for seen, _ in counts) > 0, "no copy found: the check has nothing to look at"
    assert not sum(late for _, late in counts), counts
