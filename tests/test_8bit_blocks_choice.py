"""Which kernel of the product in 8 bits with scales by blocks takes a call, on the CPU: each has the columns that it reads, whatever the sizes."""
import os
import subprocess

ONE_SCALE, SPLIT_NEAR, SPLIT_FAR, TILE, DIRECT, STAGED = range(6)
C64, F32, BF16 = (1, 1), (0, 1), (0, 0)                 # complex, results in 32 bits


def choices(tmp_path, calls):
    """(kernel, 16 rows of a wave, groups, columns needed) for (type, positions, N, K) in fields without gaps"""
    exe = str(tmp_path / "blocks_choice_check")
    source = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host", "blocks_choice_check.cpp")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", source, "-o", exe], check=True)
    lines = []
    for kind, P, N, K, apart in calls:
        v = 1 + kind[0]
        lines.append(" ".join(map(str, kind + (P * v, N, K, (P + apart) * v, P * v, P * v, 1))) + "\n")
    out = subprocess.run([exe], input="".join(lines), check=True, capture_output=True, text=True).stdout.splitlines()
    return [tuple(map(int, ln.split())) for ln in out]


def test_no_kernel_has_fewer_columns_than_it_reads(tmp_path):
    """few positions under so many rows that tiles are plenty: float32 results of 129 to 255 positions from 24449 rows on, of 128 from 49025"""
    positions = list(range(1, 300)) + [511, 512, 513, 1000, 4096, 8208, 65536, 1 << 22]
    rows = [1, 16, 17, 100, 300, 1030, 8192, 24448, 24449, 24460, 32000, 49024, 49025, 65536]
    calls = [(kind, P, N, K, apart) for kind in (C64, F32, BF16) for P in positions for N in rows for K in (1, 33, 65, 128, 256, 512, 2048, 65536) for apart in (0, 1, 1 << 27)]
    for call, (kernel, _, _, window) in zip(calls, choices(tmp_path, calls)):
        columns = call[1] * (1 + call[0][0])
        assert columns >= window, (call, kernel, window)
        assert (kernel == ONE_SCALE) == (call[3] * (1 + call[0][0]) <= 64)


def test_kernels_of_some_sizes(tmp_path):
    calls = {   # type, positions, N, K, gap -> kernel, 16 rows of a wave, groups, columns
        (BF16, 65536, 1024, 1024, 0): (DIRECT, 4, 1, 128), (BF16, 65536, 1024, 1024, 1): (STAGED, 4, 1, 128), (BF16, 1024, 1024, 1024, 0): (DIRECT, 2, 2, 128),
        (BF16, 262144, 128, 128, 0): (DIRECT, 2, 1, 128), (BF16, 2001, 1024, 1024, 0): (STAGED, 2, 2, 128), (BF16, 16, 2048, 2048, 0): (SPLIT_NEAR, 1, 1, 1),
        (BF16, 300, 100, 200, 1 << 27): (SPLIT_FAR, 1, 1, 1), (BF16, 1 << 20, 64, 64, 0): (ONE_SCALE, 0, 0, 0),
        (F32, 65536, 1024, 1024, 0): (STAGED, 4, 1, 256), (F32, 256, 24460, 200, 0): (STAGED, 4, 1, 256), (F32, 255, 24460, 200, 0): (STAGED, 2, 1, 128),
        (F32, 500, 1024, 1024, 0): (STAGED, 2, 2, 128), (F32, 128, 49200, 65, 0): (STAGED, 2, 1, 128), (F32, 127, 49200, 65, 0): (SPLIT_NEAR, 1, 1, 1),
        (C64, 30011, 136, 200, 0): (TILE, 4, 1, 64), (C64, 1024, 200, 128, 0): (TILE, 2, 1, 64), (C64, 63, 300, 128, 0): (SPLIT_NEAR, 1, 1, 1),
    }
    assert dict(zip(calls, choices(tmp_path, list(calls)))) == calls
