"""A matrix instruction's result may be used by another kind of instruction only some instructions later, and nothing in the hardware waits for
that: the compiler puts the distance in.  Where a branch comes between the two it has left it out, and the kernel read the sums of the product before.  Here every
path behind every matrix instruction of the built library is followed as far as that distance."""
import os
import re
import subprocess

import pytest

T = pytest.importorskip("tetris_amd")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
# instructions between a product and the use of its result, by the product's shape: what the compiler leaves in straight code
NEEDED = {"16x16x32": 8, "32x32x16": 12, "32x32x64": 20}
LABEL = re.compile(r"^([0-9a-f]+) <(.*)>:")
LINE = re.compile(r"^\t(\S+)\s*(.*?)\s*// ([0-9A-F]+):(.*)$")
REGISTER = re.compile(r"\b([va])\[(\d+):(\d+)\]|\b([va])(\d+)\b")


def registers(text):
    found = set()
    for kind, first, last, one, number in REGISTER.findall(text):
        found |= {(kind, i) for i in range(int(first), int(last) + 1)} if kind else {(one, int(number))}
    return found


def functions(text):
    """name, address, [(instruction, operands, address, comment)] of every function of a listing."""
    name, base, code = None, 0, []
    for line in text.split("\n"):
        m = LABEL.match(line)
        if m:
            if name:
                yield name, base, code
            name, base, code = m.group(2), int(m.group(1), 16), []
            continue
        m = LINE.match(line)
        if m and name:
            code.append((m.group(1), m.group(2), int(m.group(3), 16), m.group(4)))
    if name:
        yield name, base, code


def early_uses(base, code):
    """[(product, use, instructions between)] of uses that come too early."""
    place = {c[2]: i for i, c in enumerate(code)}

    def behind(i):
        op, _, _, comment = code[i]
        if op in ("s_endpgm", "s_setpc_b64"):
            return
        if op.startswith("s_cbranch") or op == "s_branch":
            m = re.search(r"<.*?(?:\+0x([0-9a-f]+))?>", comment)
            to = place.get(base + int(m.group(1) or "0", 16)) if m else None
            if to is not None:
                yield to
        if op != "s_branch" and i + 1 < len(code):
            yield i + 1

    found = []
    for i, (op, operands, _, _) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        needed = next(v for k, v in NEEDED.items() if k in op)
        result = registers(operands.split(",")[0])
        least, paths = {}, [(j, 0) for j in behind(i)]
        while paths:
            j, between = paths.pop()
            if between >= needed or least.get(j, needed) <= between:
                continue
            least[j] = between
            other, of, _, _ = code[j]
            if other.startswith("v_mfma"):  # (these wait for each other)
                if registers(of.split(",")[0]) >= result:
                    continue
            elif other.startswith(("v_", "ds_", "buffer_", "global_", "flat_", "scratch_")) and registers(of) & result:
                found.append((code[i][:2], code[j][:2], between))
                continue
            paths += [(k, between + (int(of.split()[0]) + 1 if other == "s_nop" else 1)) for k in behind(j)]
    return found


def test_the_search_finds_an_early_use_behind_a_branch():
    listing = """
0000000000000100 <kernel>:
\tv_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], 0 // 000000000100: D3B50000 02020D00
\ts_cbranch_vccnz 2 // 000000000108: BF870002 <kernel+0x14>
\ts_nop 7 // 00000000010C: BF800007
\tv_add_f32_e32 v9, v8, v9 // 000000000110: 02121308
\tv_accvgpr_read_b32 v8, a3 // 000000000114: D3D84008 18000103
\ts_endpgm // 00000000011C: BF810000
"""
    (name, base, code), = functions(listing)
    (product, use, between), = early_uses(base, code)
    assert name == "kernel" and use[0] == "v_accvgpr_read_b32" and between == 1
    assert not early_uses(base, [c for c in code if not c[0].startswith("s_cbranch")])


def test_no_result_of_a_matrix_instruction_is_used_too_early(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    os.symlink(T.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    kernels = 0
    for name in sorted(os.listdir(tmp_path)):
        if "gfx950" not in name or not any(k in (tmp_path / name).read_bytes() for k in (b"attend_kernel", b"tile_kernel", b"rounded_kernel", b"matrix_kernel")):
            continue
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", name], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        for symbol, base, code in functions(text):
            if any(op.startswith("v_mfma") for op, _, _, _ in code):
                kernels += 1
                early = early_uses(base, code)
                assert not early, (symbol, early[0])
    assert kernels > 50
