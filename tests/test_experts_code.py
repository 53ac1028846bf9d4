"""What the compiler made of the experts' and log-probability kernels: registers, and the wait states that it cannot see the need for."""
import os
import re
import shutil
import struct
import subprocess

import pytest

from mojo_amd import _lib
from mojo_amd.build import HIPCC

LLVM = os.path.join(os.path.dirname(os.path.dirname(HIPCC)), "llvm", "bin")
TOOLS = [os.path.join(LLVM, t) for t in ("llvm-readelf", "llvm-objcopy", "llvm-objdump")]
KERNELS = (b"experts_gemm_kernel", b"experts_small_kernel", b"logprobs_kernel", b"route_kernel")


@pytest.fixture(scope="module")
def objects(tmp_path_factory):
    """the code objects of the library that hold these kernels"""
    if not (os.path.exists(_lib.LIB_PATH) and all(map(os.path.exists, TOOLS)) and shutil.which("c++filt")):
        pytest.skip("needs the built library, llvm-readelf, llvm-objcopy, llvm-objdump and c++filt")
    tmp = tmp_path_factory.mktemp("code")
    subprocess.run([TOOLS[1], "--dump-section", f".hip_fatbin={tmp / 'fat'}", _lib.LIB_PATH, str(tmp / "rest")], check=True)
    data, found = (tmp / "fat").read_bytes(), []
    for at in (m.start() for m in re.finditer(b"__CLANG_OFFLOAD_BUNDLE__", data)):
        (entries,), p = struct.unpack_from("<Q", data, at + 24), at + 32
        for _ in range(entries):
            offset, size, length = struct.unpack_from("<QQQ", data, p)
            target = data[p + 24:p + 24 + length].decode()
            p += 24 + length
            code = data[at + offset:at + offset + size]
            if "gfx950" in target and any(k in code for k in KERNELS):
                found.append(tmp / f"{len(found)}.o")
                found[-1].write_bytes(code)
    assert len(found) == 4
    return found


def _scalars(token):
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", token)
    if m:
        return set(range(int(m[1]), int(m[2]) + 1))
    m = re.fullmatch(r"s(\d+)", token)
    return {int(m[1])} if m else set()


def _too_early(lines):
    """loads and stores that read a scalar register within five wait states of the vector instruction that wrote it"""
    function, history, found = "", [], []
    for line in lines:
        text = line.split("//")[0].strip()
        if not text:
            continue
        if text.startswith("<"):
            function, history = text, []
            continue
        op, *rest = text.split()
        tokens = [t.rstrip(",") for t in rest]
        if op.startswith(("global_", "buffer_", "flat_")):
            reads, states = set().union(*map(_scalars, tokens)) if tokens else set(), 0
            for written, waits in reversed(history):
                if states >= 5:
                    break
                if written & reads:
                    found.append((function, text, states))
                    break
                states += waits
        written = set()
        if op.startswith(("v_readfirstlane", "v_readlane", "v_cmp")) and tokens:
            written = _scalars(tokens[0])
        elif op.startswith(("v_add_co", "v_sub_co", "v_subrev_co", "v_addc", "v_subb", "v_div_scale", "v_mad_u64", "v_mad_i64")) and len(tokens) > 1:
            written = _scalars(tokens[1])
        history = (history + [(written, int(tokens[0]) + 1 if op == "s_nop" else 1)])[-8:]
    return found


def test_the_search_finds_a_load_that_is_too_early():
    code = ["<k>:", "v_readfirstlane_b32 s3, v179", "s_mov_b32 m0, s20", "s_nop 0", "global_load_lds_dwordx4 v180, s[2:3]"]
    assert len(_too_early(code)) == 1
    assert not _too_early(code[:2] + ["s_nop 4"] + code[2:]) and not _too_early(code[:4] + ["global_load_lds_dwordx4 v180, s[4:5]"])


def test_loads_in_assembly_wait_for_their_scalar_address(objects):
    """A load in inline assembly whose scalar address a vector instruction wrote just before goes to a stale address and may fault: the compiler keeps the wait states of its own loads only."""
    for o in objects:
        text = subprocess.run([TOOLS[2], "-d", "--no-show-raw-insn", "--no-leading-addr", str(o)], check=True, capture_output=True, text=True).stdout
        assert _too_early(text.splitlines()) == []


def test_nothing_is_spilled(objects):
    """Operands, sums and what is on its way are sized to a wavefront's registers; a spilled register that a load has not filled yet would be stored as it was."""
    names, spills = [], []
    for o in objects:
        notes = subprocess.run([TOOLS[0], "--notes", str(o)], check=True, capture_output=True, text=True).stdout
        for block in re.split(r"\n\s*- \.agpr_count", notes)[1:]:
            names.append(re.search(r"\n    \.name:\s+(\S+)", block).group(1))
            spills.append(int(re.search(r"\.vgpr_spill_count:\s+(\d+)", block).group(1)))
    assert len(names) > 80
    assert [n for n, s in zip(names, spills) if s and "route" not in n] == []  # (the router of more than 512 experts has no loads of its own kind)
