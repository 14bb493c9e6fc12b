"""Which blocks take which pieces of work, on the CPU: each piece is one block's, also in launches of several rows of blocks. A piece that two blocks took would be added or activated twice
where its result replaces an operand."""
import os
import subprocess

import pytest

HOST = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host")


def run(tmp_path, name, lines):
    exe = str(tmp_path / name)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", os.path.join(HOST, name + ".cpp"), "-o", exe], check=True)
    text = "".join(" ".join(map(str, ln)) + "\n" for ln in lines)
    return [tuple(map(int, ln.split())) for ln in subprocess.run([exe], input=text, check=True, capture_output=True, text=True).stdout.splitlines()]


@pytest.mark.parametrize("together", [0, 1])
def test_each_strip_is_one_block_s(tmp_path, together):
    row = 1 << 22
    strips = [1, 7, 8, 9, 64, 1000, row - 1, row, row + 1, row + 9, 2 * row, 2 * row + 2, 2 * row + 17]
    assert run(tmp_path, "block_order_check", [(0, n, together) for n in strips]) == [(0, 0)] * len(strips)


@pytest.mark.parametrize("turns", [0, 1])
def test_each_tile_is_one_block_s(tmp_path, turns):
    row = 1 << 22
    tiles = [(1, 1), (3, 63), (3, 64), (2, 65), (17, 1001), (1, row - 7), (1, row), (1, row + 1), (1, row + 9), (3, row // 3), (3, row // 3 + 5), (5, row // 2 + 3), (1024, 4095), (1024, 4097)]
    assert run(tmp_path, "block_order_check", [(1,) + t + (turns,) for t in tiles]) == [(0, 0)] * len(tiles)


@pytest.mark.parametrize("together", [0, 1])
def test_strips_of_the_layer_norm_s_gradient(tmp_path, together):
    """each strip is one block's, no block has more than 64 of a launch, or 65 where eighths do not come out even, and the workspace has room for the blocks of all launches"""
    columns = [1, 7, 8, 9, 500, 4095, 4096, 8191, 8192, 30011, 1 << 16, 131080, (1 << 20) - 1, 1 << 20, (1 << 20) + 1, (1 << 21) + 32, (1 << 21) + 33, 3000001, (1 << 22) + 4096 * 3 + 1, 1 << 23,
               (1 << 23) + 1, 50000003, (1 << 26) + 33, 1 << 28]
    calls = [(2, n, lanes, together) for n in columns for lanes in ((64, 16, 8) if n >= 8192 else (64, 16, 8, 4, 2))]
    out = run(tmp_path, "block_order_check", calls)
    assert len(out) == 2 * len(calls)
    for call, strips, (most, blocks, room) in zip(calls, out[::2], out[1::2]):
        assert strips == (0, 0) and most <= 64 + together and blocks <= room, (call, strips, most, blocks, room)
