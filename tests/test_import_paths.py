"""Both import paths reach everything that trains the gated layer, its update too."""

import pathlib
import subprocess
import sys

ROOT = pathlib.Path(__file__).resolve().parents[1]


def test_the_update_is_reached_by_the_reference_s_import_path() -> None:
    code = ("from sparsebench import moe, optim; import sparsebench.optim, sparsebench_amd.optim as own; "
            "assert sparsebench.optim is own is optim; moe.moe_gated_train, optim.AdamW, optim.adamw_step")
    subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True, capture_output=True, timeout=300)
