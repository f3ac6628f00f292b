"""CPU check of the metadata of the library built here: the kernels of linear attention and of the block join take no
private memory. A kernel that spills registers gets it from the runtime, which allocates for as many waves as the
card holds when such a kernel is first launched: inside a call that is to allocate nothing."""

import os
import re
import shutil
import subprocess

import pytest

from test_isa import LLVM, MAGIC, TARGET
from zenjpegai_amd import _lib


def private_bytes(so_path, folder):
    """{kernel: bytes of private memory of a lane} of the library's kernels."""
    lib, fat, out = (os.path.join(folder, n) for n in ("lib.so", "fat", "object"))
    shutil.copyfile(so_path, lib)
    subprocess.run(["objcopy", "--dump-section", f".hip_fatbin={fat}", lib, "/dev/null"], capture_output=True, check=True)
    data = open(fat, "rb").read()
    starts = [m.start() for m in re.finditer(re.escape(MAGIC), data)] + [len(data)]
    sizes = {}
    for a, b in zip(starts, starts[1:]):
        with open(fat, "wb") as f:
            f.write(data[a:b])
        subprocess.run([f"{LLVM}/clang-offload-bundler", "--type=o", f"--targets={TARGET}", f"--input={fat}", f"--output={out}",
                        "--unbundle"], capture_output=True, check=True)
        notes = subprocess.run([f"{LLVM}/llvm-readelf", "--notes", out], capture_output=True, text=True, check=True).stdout
        names = re.findall(r"^ {4}\.name: +(\S+)$", notes, re.M)
        private = re.findall(r"^ {4}\.private_segment_fixed_size: (\d+)$", notes, re.M)
        assert len(names) == len(private)
        sizes.update(zip(names, map(int, private)))
    return sizes


@pytest.mark.skipif(not (shutil.which("objcopy") and os.path.exists(f"{LLVM}/llvm-readelf")), reason="ROCm LLVM tools not installed")
def test_kernels_of_calls_that_allocate_nothing_take_no_private_memory(tmp_path):
    sizes = private_bytes(_lib.LIB_PATH, str(tmp_path))
    mine = {k: v for k, v in sizes.items() if "k_linear_" in k or "k_join" in k}
    assert len(mine) >= 130, len(mine)
    assert not any(mine.values()), {k: v for k, v in mine.items() if v}
