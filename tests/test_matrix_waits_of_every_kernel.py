"""The search of test_matrix_waits over every kernel of the built library that has matrix instructions, whatever its name and object, sparse products among
them; and the kernels that have to be among those searched, so that a renamed one is missed here."""
import os
import re
import subprocess

import pytest

import test_matrix_waits as W

T = pytest.importorskip("tetris_amd")
PRODUCTS = ("v_mfma", "v_smfmac")
# a sparse product of 32x32x32 takes as long as a dense one of 32x32x16
NEEDED = {**W.NEEDED, "32x32x32": 12}
SEARCHED = {"attend_chunks_kernel", "attend_shares_kernel", "attend_prompt_kernel", "tile_kernel", "rounded_kernel", "stream_kernel", "down_kernel", "matrix_kernel",
            "half_kernel"}


def products(code):
    """The instructions with sparse products named as dense ones, which is how the search knows them; and whether there are any of either."""
    named = [(op.replace("v_smfmac", "v_mfma"), *rest) for op, *rest in code]
    return named, any(op.startswith("v_mfma") for op, *_ in named)


def kernel_of(symbol):
    """The last of the names in a nested mangled name (_ZN, then each name behind its length)."""
    at, name = len("_ZN") if symbol.startswith("_ZN") else len(symbol), symbol
    while at < len(symbol) and symbol[at].isdigit():
        length = re.match(r"\d+", symbol[at:]).group()
        at += len(length)
        name = symbol[at:at + int(length)]
        at += int(length)
    return name


def test_an_early_use_of_a_sparse_product_is_found(monkeypatch):
    monkeypatch.setattr(W, "NEEDED", NEEDED)
    listing = """
0000000000000100 <_ZN6tetris12_GLOBAL__N_111half_kernelILi1EEEvi>:
\tv_smfmac_f32_32x32x32_f16 v[0:15], v[16:19], v[20:27], v28 // 000000000100: D3D40000 02020D00
\ts_cbranch_vccnz 2 // 000000000108: BF870002 <_ZN6tetris12_GLOBAL__N_111half_kernelILi1EEEvi+0x18>
\ts_nop 7 // 00000000010C: BF800007
\ts_nop 3 // 000000000110: BF800003
\ts_nop 0 // 000000000114: BF800000
\tv_mul_f32_e32 v30, v3, v31 // 000000000118: 0A3C3F03
\ts_endpgm // 00000000011C: BF810000
"""
    (symbol, base, code), = W.functions(listing)
    named, any_product = products(code)
    assert kernel_of(symbol) == "half_kernel" and any_product
    (_, use, between), = W.early_uses(base, named)
    assert use[0] == "v_mul_f32_e32" and between == 1
    assert not W.early_uses(base, [c for c in named if not c[0].startswith("s_cbranch")])


def test_no_result_is_used_too_early_in_any_kernel(tmp_path, monkeypatch):
    if not os.path.exists(W.OBJDUMP):
        pytest.skip("no llvm-objdump")
    monkeypatch.setattr(W, "NEEDED", NEEDED)
    os.symlink(T.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([W.OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    searched = set()
    for name in sorted(os.listdir(tmp_path)):
        if "gfx950" not in name:
            continue
        text = subprocess.run([W.OBJDUMP, "-d", "--no-show-raw-insn", name], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        if not any(p in text for p in PRODUCTS):
            continue
        for symbol, base, code in W.functions(text):
            code, any_product = products(code)
            if not any_product:
                continue
            unknown = {op for op, *_ in code if op.startswith("v_mfma") and not any(shape in op for shape in NEEDED)}
            assert not unknown, "how long these take is not known here: %s" % unknown
            early = W.early_uses(base, code)
            assert not early, (symbol, early[0])
            searched.add(kernel_of(symbol))
    assert SEARCHED <= searched, SEARCHED - searched
