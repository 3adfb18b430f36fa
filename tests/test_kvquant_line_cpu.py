"""How attention over the 8-bit cache is cut over CTAs (csrc/kvquant_line.h), walked on the CPU over batches, heads, grids and lengths."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_no_two_sums_share_a_ticket_and_no_two_pieces_a_slot(tmp_path):
    exe = str(tmp_path / "walk")
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", os.path.join(HERE, "..", "denograd_b200", "csrc"), os.path.join(HERE, "kvquant_line_walk.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
