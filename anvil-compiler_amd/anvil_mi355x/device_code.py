"""What the compiler may not leave in a library's device code: a 64-bit shift by the last vector register of its kernel.

On the MI355X v_lshlrev_b64, v_lshrrev_b64 and v_ashrrev_i64 now and then shift by another amount, one of its own in every lane, if their amount
stands in the last vector register that the wave has been given (number 8 n + 7, with nothing behind it) and other waves come and go on the SIMD. The
compiler (ROCm 7.2) knows this of an older generation and does not keep off it here. Measured on a kernel of 48 registers that shifts by v47, 140003
rows of 32 lanes: 8 to 12 thousand lanes were wrong, 90 to 108 thousand with idle cycles between write and shift, none with 56 or 64 registers or
with the amount copied to another register first. v_ldexp_f64, v_mad_u64_u32, v_mad_i64_i32, v_trig_preop_f64, v_cmp_class_f64 and the conversions to
64 bits read the same register rightly. A kernel that is named here needs some change of its registers, such as one more that it keeps.
"""
from __future__ import annotations

import re
import struct
import subprocess
import tempfile
from pathlib import Path

LLVM = Path("/opt/rocm/llvm/bin")
BUNDLE = b"__CLANG_OFFLOAD_BUNDLE__"
SHIFT = re.compile(r"\s+v_(?:lshlrev_b64|lshrrev_b64|ashrrev_i64)\S* v\[\d+:\d+\], v(\d+),")


def code_objects(path) -> list[bytes]:
    """The device code objects of a library or an object file."""
    data, found, at = Path(path).read_bytes(), [], -1
    while (at := data.find(BUNDLE, at + 1)) >= 0:
        entries, entry = struct.unpack_from("<Q", data, at + len(BUNDLE))[0], at + len(BUNDLE) + 8
        for _ in range(entries):
            offset, size, length = struct.unpack_from("<QQQ", data, entry)
            if size and b"amdgcn" in data[entry + 24:entry + 24 + length]:
                found.append(data[at + offset:at + offset + size])
            entry += 24 + length
    return found


def _run(tool, *args):
    return subprocess.run([str(LLVM / tool), *args], capture_output=True, text=True, check=True).stdout


def _last_registers(notes) -> dict:
    """{kernel: number of its last vector register}: they come in eights, with accumulation registers in fours before those."""
    last = {}
    for kernel in notes.split("- .agpr_count:")[1:]:
        acc, name = int(kernel.split()[0]), re.search(r"\.symbol:\s+(\S+)\.kd", kernel).group(1)
        total = int(re.search(r"\.vgpr_count:\s+(\d+)", kernel).group(1))
        last[name] = (total - acc + 3) // 4 * 4 - 1 if acc else (total + 7) // 8 * 8 - 1
    return last


def last_register_shifts(path) -> list[str]:
    """The 64-bit shifts by a kernel's last vector register, "kernel: instruction" each; of a function that kernels share, those by any that may be."""
    objects, found = code_objects(path), []
    if not objects:
        raise RuntimeError(f"{path}: no device code found")
    with tempfile.TemporaryDirectory() as tmp:
        for n, code in enumerate(objects):
            obj = Path(tmp, f"{n}.co")
            obj.write_bytes(code)
            last, name = _last_registers(_run("llvm-readelf", "--notes", str(obj))), ""
            for line in _run("llvm-objdump", "-d", "--no-show-raw-insn", str(obj)).splitlines():
                if m := re.match(r"[0-9a-f]+ <(\S+)>:", line):
                    name = m.group(1)
                elif m := SHIFT.match(line):
                    v = int(m.group(1))
                    if v == last[name] if name in last else v % 8 == 7:
                        found.append(f"{name}: {line.split('//')[0].strip()}")
    return found
