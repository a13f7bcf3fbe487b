"""The kernels of MX4 products wait for loads by their number (csrc/mx4_product.hip, barrier_but): all that were issued but the last N.  That is
right only if loads are issued in the order that the count assumes, which is looked at here in the built library."""
import os
import re
import subprocess

import pytest

T = pytest.importorskip("tetris_amd")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


@pytest.fixture(scope="module")
def prologues(tmp_path_factory):
    """By kernel: its vector loads up to the first barrier in order, "rows" for those to LDS, and the number that the barrier's wait leaves under way."""
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    d = tmp_path_factory.mktemp("code")
    os.symlink(T.LIB_PATH, d / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=d, check=True, capture_output=True)
    name = next(f for f in sorted(os.listdir(d)) if "gfx950" in f and b"rounded_kernel" in (d / f).read_bytes())
    text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", name], cwd=d, check=True, capture_output=True, text=True).stdout
    found = {}
    for part in re.split(r"^[0-9a-f]+ <", text, flags=re.M)[1:]:
        symbol = part[:part.index(">")]
        if "tile_kernel" not in symbol and "rounded_kernel" not in symbol:
            continue
        loads, left = [], None
        for line in part.split("\n"):
            line = line.split("//")[0].strip()
            if line.startswith(("buffer_load", "global_load")):
                loads.append("rows" if line.endswith(" lds") else "weights" if line.startswith("buffer") else "index")
            elif line.startswith("s_waitcnt") and "vmcnt" in line:
                left = int(re.search(r"vmcnt\((\d+)\)", line).group(1))
            elif line.startswith("s_barrier"):
                break
        found[symbol] = loads, left
    return found


def test_rounded_kernel_asks_for_rows_and_weights_step_by_step(prologues):
    kernels = {k: v for k, v in prologues.items() if "rounded_kernel" in k}
    assert len(kernels) == 3  # a type of output each
    for loads, left in kernels.values():
        # three steps: two loads of rows a wave, then three of each of two tiles of weights and one of each of four tiles of rows' scales
        assert loads == (["rows"] * 2 + ["weights"] * 10) * 3
        assert left == len(loads) - 2  # the first step's rows have arrived


def test_tile_kernel_asks_for_rows_last(prologues):
    kernels = {k: v for k, v in prologues.items() if "tile_kernel" in k}
    assert len(kernels) > 20
    for symbol, (loads, left) in kernels.items():
        first = loads.index("rows")
        rows = loads[first:]
        assert set(rows) == {"rows"}, symbol  # nothing comes between them
        assert "weights" in loads[:first] and len(rows) == 2 * left, symbol  # two steps; the first has arrived
