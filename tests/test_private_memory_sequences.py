"""CPU: the kernels of rotary positions, the causal convolution and the selective scan have no private memory, which the runtime would
take from the card in calls that allocate nothing."""

import os
import shutil

import pytest

from test_private_memory import LLVM, private_bytes
from zenjpegai_amd import _lib


@pytest.mark.skipif(not (shutil.which("objcopy") and os.path.exists(f"{LLVM}/llvm-readelf")), reason="ROCm LLVM tools not installed")
def test_kernels_on_sequences_take_no_private_memory(tmp_path):
    sizes = private_bytes(_lib.LIB_PATH, str(tmp_path))
    mine = {k: v for k, v in sizes.items() if "k_rotary" in k or "k_causal_conv" in k or "k_scan" in k}
    assert len(mine) >= 200, len(mine)
    assert not any(mine.values()), {k: v for k, v in mine.items() if v}
