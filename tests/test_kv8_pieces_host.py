"""Where the workgroups of a long extension over caches held in 8 bits find their work
(``csrc/kv8_pieces.h``), for offsets and contexts of any contents, on the host."""

import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_pieces_of_any_offsets_stay_in_range(tmp_path):
    """Rows that overlap can cost more than 32 bits hold; no piece, unit, slot, partial or join is out of range."""
    exe = tmp_path / "walk"
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", os.path.join(HERE, "kv8_pieces_walk.cpp"), "-o", exe],
                   check=True)
    run = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout
