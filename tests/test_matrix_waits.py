"""Wait states between the matrix products of csrc/kernels/paged.hip and what
reads their results, in the code object that the build made of it.

gfx950 does not hold an instruction back that reads a product's result: the
code has to let wait states pass, 8 behind a 16 x 16 product of 4 passes (halves
and bf16) and 10 behind one of 8 (single), which is what the compiler leaves
where nothing lies between the two. It counts them along the code as it is laid
out, and has been seen to miss the shorter way round a block that is skipped
when no lane needs it. Here every way is followed."""
import os
import re
import struct
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OBJECT = os.path.join(ROOT, "mormot2-ai_amd", "_build", "paged.hsaco")
OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")
WAITS = {"v_mfma_f32_16x16x4_f32": 10, "v_mfma_f32_16x16x32_f16": 8, "v_mfma_f32_16x16x32_bf16": 8}


def registers(text):
    out = set()
    for file, lo, hi, one, at in re.findall(r"\b([va])\[(\d+):(\d+)\]|\b([va])(\d+)\b", text):
        out |= {(file, i) for i in range(int(lo), int(hi) + 1)} if file else {(one, int(at))}
    return out


def parse(lines):
    """[(instruction, index of the branch's target or None)] of one function's listing."""
    code, at = [], {}
    for line in lines:
        m = re.match(r"\s+(\S.*?)\s*//\s*([0-9A-Fa-f]+):(?:.*<[^+>]+(?:\+0x([0-9a-fA-F]+))?>)?", line)
        if m:
            at[int(m.group(2), 16)] = len(code)
            code.append((m.group(1), int(m.group(3) or "0", 16) if "branch" in m.group(1) else None))
    start = min(at) if at else 0
    return [(i, None if t is None else at[start + t]) for i, t in code]


def too_soon(code):
    """The (product, reader, wait states between) that come too soon, on any way."""
    found = []
    for i, (text, _) in enumerate(code):
        if not text.startswith("v_mfma"):
            continue
        result, waits = registers(text.split(",")[0]), WAITS[text.split()[0]]
        ways, best = [(i + 1, 0)], {}
        while ways:
            j, waited = ways.pop()
            if j >= len(code) or waited >= waits or best.get(j, waits) <= waited:
                continue
            best[j] = waited
            x, target = code[j]
            op, _, args = x.partition(" ")
            if op.startswith("v_mfma"):  # (sums follow each other without a wait; factors do not)
                args = ",".join(args.split(",")[1:3])
            if not op.startswith("s_") and registers(args) & result:
                found.append((text, x, waited))
                break
            if op in ("s_endpgm", "s_setpc_b64"):
                continue
            # (a sleep of 64 clocks is 16 wait states of 4)
            waited += int(args, 0) + 1 if op == "s_nop" else 16 * int(args, 0) if op == "s_sleep" else 1
            if target is not None:
                ways.append((target, waited))
                if op == "s_branch":
                    continue
            ways.append((j + 1, waited))
    return found


def listing(*lines):
    return parse([f"\t{text} // {4 * i:012X}: 00000000{f' <k+0x{4 * to:x}>' if to is not None else ''}"
                  for i, (text, to) in enumerate(lines)])


def test_the_check_itself():
    product = ("v_mfma_f32_16x16x4_f32 v[0:3], v8, v9, v[0:3]", None)
    reader, other = ("v_mul_f32_e32 v4, v3, v5", None), ("v_mul_f32_e32 v6, v7, v5", None)
    assert too_soon(listing(product, ("s_nop 9", None), reader)) == []
    assert len(too_soon(listing(product, ("s_nop 8", None), reader))) == 1
    assert len(too_soon(listing(product, other, reader))) == 1
    assert too_soon(listing(product, product, other, ("s_endpgm", None), reader)) == []
    # the block that may be skipped holds the waits
    skipped = [product, ("s_cbranch_execz 15", 4), ("s_nop 15", None), other, reader]
    assert len(too_soon(listing(*skipped))) == 1
    skipped[1:3] = [("s_nop 15", None), ("s_cbranch_execz 15", 4)]
    assert too_soon(listing(*skipped)) == []
    # round a loop: read at its head in the next turn
    loop = [reader, other, product, ("s_cbranch_scc1 65532", 0), ("s_endpgm", None)]
    assert len(too_soon(listing(*loop))) == 1
    assert too_soon(listing(product, ("s_sleep 1", None), reader)) == []
    assert len(too_soon(listing(product, ("s_sleep 0", None), reader))) == 1
    # a result as the next product's factor, as its sum
    assert len(too_soon(listing(product, ("v_mfma_f32_16x16x4_f32 v[12:15], v1, v9, v[12:15]", None)))) == 1
    assert too_soon(listing(product, product)) == []


@pytest.mark.skipif(not os.path.exists(OBJECT) or not os.path.exists(OBJDUMP), reason="no code object or disassembler")
def test_products_of_the_paged_kernels(tmp_path):
    # the bundle that the build makes holds a table of (start, size, name's length, name)
    with open(OBJECT, "rb") as f:
        bundle = f.read()
    at, part = 32, None
    for _ in range(struct.unpack_from("<Q", bundle, 24)[0]):
        start, size, name = struct.unpack_from("<QQQ", bundle, at)
        if size and b"gfx950" in bundle[at + 24:at + 24 + name]:
            part = bundle[start:start + size]
        at += 24 + name
    (tmp_path / "paged.elf").write_bytes(part)
    text = subprocess.run([OBJDUMP, "-d", str(tmp_path / "paged.elf")], capture_output=True, text=True, check=True).stdout
    kernels = {}
    for line in text.splitlines():
        m = re.match(r"[0-9a-f]+ <(\w+)>:", line)
        if m:
            body = kernels.setdefault(m.group(1), [])
        elif kernels:
            body.append(line)
    seen = 0
    for name, lines in kernels.items():
        code = parse(lines)
        seen += sum(i.startswith("v_mfma") for i, _ in code)
        assert too_soon(code) == [], name
    assert sum(n.startswith("paged_attention") for n in kernels) == 24 and seen > 24 * 8
