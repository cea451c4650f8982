"""What the bulk-copy kernels of page copies and compaction leave behind when a wait gives up, on emulated lanes."""

import pathlib
import re
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    source = (ROOT / "turboquant-vllm_b200" / "csrc" / "tq4_rows.cu").read_text()
    constants, rest = source.split("constexpr int kMaxLayers", 1)[1].split("__device__ __forceinline__ uint32_t smem_of", 1)
    kernels = rest.split("// Pages copied", 1)[1].split("// Largest piece", 1)[0]
    text = "constexpr int kMaxLayers" + constants + "// Pages copied" + kernels
    text = re.sub(r"extern __shared__ __align__\(128\) unsigned char s_rows\[\];", "unsigned char* s_rows = g_rows;", text)
    text = re.sub(r"asm volatile\(.*\);", ";", text)  # (loads of the kernel without bulk copies, which is not run)
    folder = tmp_path_factory.mktemp("emulated")
    (folder / "rows.inc").write_text(text)
    here = ROOT / "tests" / "emulated"
    subprocess.run(["g++", "-std=c++20", "-O1", "-w", "-pthread", f"-I{here}", f"-I{folder}", f"-I{ROOT / 'include'}",
                    str(here / "rows_give_up.cpp"), "-o", str(folder / "rows_give_up")], check=True)
    return folder / "rows_give_up"


@pytest.mark.parametrize("kernel", ["pages", "short", "long"])
def test_a_wait_that_gives_up_loses_no_row_and_leaves_no_copy_in_flight(program, kernel):
    done = subprocess.run([str(program), kernel], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout + done.stderr
