"""The bytes that the paged attention reads of a key or value row, checked on the CPU: the kernel forms them by
the functions of vkernels_amd/csrc/paged_attention_layout.hpp, and tests/paged_attention_layout_check.cpp
(compiled here with g++) walks all lanes and loads with the same functions.  Rows of 96 and 192 values have
fewer pieces than the lanes that load them: such a lane must not read behind the row, which may be the last
of the cache's memory."""
from __future__ import annotations

import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "vkernels_amd" / "csrc"


def _compiled(into, include):
    exe = into / "paged_attention_layout_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", f"-I{include}",
                    str(ROOT / "tests" / "paged_attention_layout_check.cpp"), "-o", str(exe)], check=True)
    return exe


@pytest.fixture(scope="module")
def checker(tmp_path_factory):
    return _compiled(tmp_path_factory.mktemp("layout"), CSRC)


@pytest.mark.parametrize("elem", [1, 2])
@pytest.mark.parametrize("D", range(16, 257, 16))
def test_no_lane_reads_outside_a_row(checker, D, elem):
    res = subprocess.run([str(checker), str(D), str(elem)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr.strip()


def test_the_kernel_reads_rows_through_the_checked_functions():
    src = (CSRC / "paged_attention.hip").read_text()
    assert "const uint32_t value_at = pa_value_at(piece, row_bytes);" in src
    assert "row + pa_piece_at(at, row_bytes)" in src
    assert "const int row_bytes = FULL ? L::kRowBytes : a.D * L::kElem;" in src


@pytest.mark.parametrize("D,elem", [(96, 2), (192, 1), (192, 2), (80, 2)])
def test_the_checker_notices_reads_behind_a_row(tmp_path, D, elem):
    """Pieces dealt out to all lanes of a row, whether it has them or not."""
    src = (CSRC / "paged_attention_layout.hpp").read_text()
    kept = "{ return at < row_bytes ? at : 0; }"
    assert kept in src
    (tmp_path / "paged_attention_layout.hpp").write_text(src.replace(kept, "{ return row_bytes > 0 ? at : 0; }"))
    res = subprocess.run([str(_compiled(tmp_path, tmp_path)), str(D), str(elem)], capture_output=True, text=True)
    assert res.returncode == 1 and "reads [" in res.stderr
