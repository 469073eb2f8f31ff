"""The operators for language models on the checked build of the library (index checks inside the kernels,
-DHC_CUDA_CHECKED) on a B200: their tests run with the checks compiled in, and none fires."""

from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

REPO = Path(__file__).resolve().parent.parent
CHECKED = REPO / "5_b200" / "lib" / "libhc_cuda_checked.so"


@pytest.mark.parametrize("module, some", [
    ("test_gpu_norm.py", "test_many_rows or test_pitches or test_a_window"),
    ("test_gpu_linear_loss.py", "test_loss_and_gradients or test_pieces or test_long_sums"),
    ("test_gpu_gemm_w4.py", "test_products or test_blocks or test_pitches or test_weights"),
])
def test_the_operators_pass_their_checks(module, some) -> None:
    assert CHECKED.exists(), "build it with `python 5_b200/build.py --checked`"
    code = ("import sys, pytest; from hc import cuda; assert cuda.library_is_checked(); "
            "sys.exit(pytest.main(sys.argv[1:]))")
    env = dict(os.environ, HC_CUDA_LIB=str(CHECKED),
               PYTHONPATH=os.pathsep.join([str(REPO / "5_b200"), os.environ.get("PYTHONPATH", "")]))
    done = subprocess.run([sys.executable, "-c", code, str(REPO / "tests" / module), "-x", "-q", "-m", "gpu", "-k", some,
                           "-p", "no:cacheprovider"], env=env, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stdout[-3000:] + done.stderr[-2000:]
