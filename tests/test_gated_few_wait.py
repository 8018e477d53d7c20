"""The sum that the last workgroup of few_down_kernel makes of the others'
results (csrc/gated_few.hip): every wave has its stores written before the
workgroup's barrier, after which one lane writes the cache back and draws the
ticket. A barrier alone does not wait for other waves' stores on gfx950, so
the wait is looked for in the assembly of the kernels, on the CPU."""

import re
import subprocess

import pytest
import torch

from sparsebench_amd import build


def kernels(assembly: str) -> dict[str, list[str]]:
    found = {}
    for m in re.finditer(r"^(\w*few_down_kernel\w*):", assembly, re.M):
        lines = assembly[m.end():assembly.index(".Lfunc_end", m.end())].splitlines()
        found[m.group(1)] = [text for line in lines if (text := line.split(";")[0].strip())]
    return found


def waits_before_ticket(lines: list[str]) -> bool:
    """Whether each wave's memory operations are waited for in a straight line before the ticket's barrier."""
    ticket = next(i for i, line in enumerate(lines) if line.startswith("global_atomic_add"))
    at = max(i for i in range(ticket) if lines[i].startswith("s_barrier"))
    for line in reversed(lines[:at]):
        if line.startswith("s_waitcnt") and "vmcnt(0)" in line:
            return True
        if line.startswith(("global_", "buffer_", "flat_", "s_cbranch", "s_branch", ".L")):
            return False
    return False


def test_every_wave_waits_for_its_stores_before_the_ticket(tmp_path) -> None:
    try:
        hipcc = build.hipcc()
    except RuntimeError as e:
        pytest.skip(str(e))
    out = tmp_path / "few.s"
    subprocess.run([hipcc, *build.HIPCC_FLAGS, "-S", "--cuda-device-only", str(build.CSRC / "gated_few.hip"), "-o",
                    str(out)], check=True, capture_output=True)
    drawing = {name: lines for name, lines in kernels(out.read_text()).items()
               if any(line.startswith("global_atomic_add") for line in lines)}
    assert len(drawing) == 4  # one or two tokens, two activations
    for name, lines in drawing.items():
        assert waits_before_ticket(lines), name


@pytest.mark.gpu
@pytest.mark.parametrize(("t", "k", "d", "f"), [(1, 2, 256, 512), (2, 2, 256, 512), (1, 1, 128, 2048), (2, 4, 128, 256)])
def test_no_workgroup_reads_another_s_sums_too_early(t, k, d, f) -> None:
    """The workspace holds NaN before each of many calls, which any sum read too early would be."""
    from sparsebench_amd import _C
    from sparsebench_amd._lib import check, lib, stream_of
    from tests.test_gated_gpu import make

    x, idx, gates, w1, w2, _ = (v.cuda() for v in make(t, k, 8, d, f, seed=t + d))
    size = _C.gated_bytes(t, k, 8, d, f)[0]
    workspace = torch.empty(size // 4, dtype=torch.float32, device="cuda")
    outs = torch.zeros(300, t, d, dtype=torch.bfloat16, device="cuda")
    for out in outs:
        workspace.fill_(float("nan"))
        check(lib().sb_gated_layer(x.data_ptr(), idx.data_ptr(), 1, gates.data_ptr(), 0, w1.data_ptr(), w2.data_ptr(),
                                   out.data_ptr(), 0, workspace.data_ptr(), size, t, k, 8, d, f, None,
                                   stream_of(x.device)))
    assert torch.isfinite(outs.float()).all() and bool((outs == outs[0]).all())
