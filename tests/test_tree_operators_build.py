"""Tree attention: what its kernels take for granted about every width of heads, asked of the compiler."""
import subprocess

import pytest

from logismos_amd import build

WIDTHS = [32, 64, 96, 128, 160, 192, 224, 256]


def test_operands_are_read_ahead_as_far_as_there_are_any(tmp_path):
    """A head of 32 has two matrix operands a product: a third one read ahead would lie outside the arrays and the tile."""
    try:
        exe = build.hipcc()
    except RuntimeError:
        pytest.skip("no hipcc")
    src = tmp_path / "lead.hip"
    src.write_text('#include "paged_attn_tree.hpp"\n' + "".join(
        f'static_assert(lg::tree_steps({d}) == {d} / 16 && lg::tree_lead({d}) >= 1 && '
        f'lg::tree_lead({d}) <= lg::tree_steps({d}), "heads of {d}");\n' for d in WIDTHS))
    r = subprocess.run([exe, "-fsyntax-only", "--cuda-host-only", f"--offload-arch={build.OFFLOAD_ARCH}", "-std=c++17",
                        "-Wno-everything", "-I", build.CSRC, "-x", "hip", str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
