"""The listings of the code objects that the build made (for the checks of wait states)."""
import os
import re
import struct
import subprocess

from test_matrix_waits import OBJDUMP, ROOT, parse, too_soon


def build_of(name):
    return os.path.join(ROOT, "mormot2-ai_amd", "_build", name + ".hsaco")


def kernels(name, folder):
    """{kernel: its instructions} of a code object of the build."""
    # the bundle holds a table of (start, size, name's length, name)
    with open(build_of(name), "rb") as f:
        bundle = f.read()
    at, part = 32, None
    for _ in range(struct.unpack_from("<Q", bundle, 24)[0]):
        start, size, n = struct.unpack_from("<QQQ", bundle, at)
        if size and b"gfx950" in bundle[at + 24:at + 24 + n]:
            part = bundle[start:start + size]
        at += 24 + n
    elf = folder / (name + ".elf")
    elf.write_bytes(part)
    text = subprocess.run([OBJDUMP, "-d", str(elf)], capture_output=True, text=True, check=True).stdout
    out = {}
    for line in text.splitlines():
        m = re.match(r"[0-9a-f]+ <(\w+)>:", line)
        if m:
            body = out.setdefault(m.group(1), [])
        elif out:
            body.append(line)
    return {k: parse(lines) for k, lines in out.items()}


def products_wait(name, folder):
    """Every product of every kernel waits before its result is read; how many products."""
    seen = 0
    for kernel, code in kernels(name, folder).items():
        seen += sum(i.startswith("v_mfma") for i, _ in code)
        assert too_soon(code) == [], kernel
    return seen
