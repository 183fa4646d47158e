"""Launches and allocations of the training entries over the sizes that they accept, on the host (tests/host_runtime.py: no kernel runs)."""
import pytest

from tests import host_runtime


@pytest.fixture
def host(tmp_path_factory):
    return lambda script: host_runtime.run(tmp_path_factory, _CALLS + script)


_CALLS = """
P = 1 << 40
def norm(rows, cols, stream=0):
    return lib.qgemm_layer_norm(BF16, BF16, F32, I8, P, cols, P, P, 1e-5, P, cols, P, P, P, cols, P, rows, cols, stream)
def backward(rows, cols, stream=0, dweight=P, x=BF16):
    return lib.qgemm_layer_norm_backward(BF16, x, BF16, F32, P, cols, P, cols, P, P, P, P, P, cols, dweight, dweight, rows, cols, stream)
def checkpoint(rows, cols, stream=0):
    return lib.qgemm_checkpoint(BF16, I8, P, cols, rows, cols, P, cols, P, stream)
def restore(rows, cols, stream=0):
    return lib.qgemm_restore(I8, BF16, P, cols, P, rows, cols, P, cols, stream)
def gradient(rows, n, cols, stream=0):
    return lib.qgemm_weight_gradient(BF16, I8, F32, F32, P, n, P, cols, P, P, P, P, cols, P, rows, n, cols, stream)
OK, TOO_LARGE = 0, 9
def launches():
    out = []
    for e in events():
        m = re.match(r"launch _ZN5qgemm[0-9]+([a-z0-9_]+?_kernel).* grid ([0-9]+) ([0-9]+) block ([0-9]+)", e)
        if m:
            out.append((m[1], *map(int, m.groups()[1:])))
    return out
"""


def test_no_launch_is_larger_than_the_runtime_takes(host):
    """Fewer than 2^32 threads across and 2^16 workgroups down, whatever size is not refused."""
    host("""
import random
rng = random.Random(1)
runtime.host_budget(1 << 62)
def check(what, status):
    made = launches()
    assert status in (OK, TOO_LARGE) and bool(made) == (status == OK), (what, status, made)
    for name, x, y, block in made:
        assert 0 < x * block < 1 << 32 and 0 < y < 1 << 16, (what, name, x, y, block)
edges = [1, 7, 8, 16384, 16385, 1 << 18, 1 << 24, 1 << 27, (1 << 28) - 33, (1 << 28) - 31, 1 << 28, (1 << 28) + 5, 1 << 30, (1 << 31) - 129, (1 << 31) - 128, (1 << 31) - 127,
         (1 << 31) - 1, 1 << 31]
size = lambda: rng.choice(edges) if rng.random() < 0.3 else int(2 ** rng.uniform(0, 31))
for _ in range(3000):
    rows, cols = size(), size()
    check(("norm", rows, cols), norm(rows, cols))
    check(("backward", rows, cols), backward(rows, cols))
    check(("backward out of codes", rows, cols), backward(rows, cols, x=I8))
    check(("checkpoint", rows, cols), checkpoint(rows, cols))
    check(("restore", rows, cols), restore(rows, cols))
    n = size()
    check(("gradient", rows, n, cols), gradient(rows, n, cols))
assert backward(3, 1 << 28) == OK and backward(0, (1 << 31) - 128) == OK
""")


def test_partial_sums_stay_within_their_room(host):
    """Sums of columns that pass through the workspace: 128 MiB at the most, or the eight bytes a column that one part of them takes."""
    host("""
import random
rng = random.Random(2)
runtime.host_budget(1 << 62)
def most():
    sizes = [int(e.split()[1]) for e in events() if e.startswith("malloc")]
    return max(sizes, default=0)
for rows, cols in [(1009, 1 << 18), (5000, (1 << 18) + 1), (70000, 1 << 20), (1 << 20, 16384), (16, 1 << 24), (17, 1 << 24), (3000, 1 << 28)] + \
                  [(int(2 ** rng.uniform(0, 20)), int(2 ** rng.uniform(0, 28))) for _ in range(500)]:
    lib.qgemm_shutdown()
    events()
    assert backward(rows, cols) == OK
    took = most()
    assert took <= max(128 << 20, 8 * ((cols + 63) // 64 * 64)), (rows, cols, took)
    lib.qgemm_shutdown()
    events()
    assert backward(rows, cols, dweight=None) == OK and most() == 0
    n, cols = int(2 ** rng.uniform(0, 14)), int(2 ** rng.uniform(0, 14))
    assert gradient(rows, n, cols) == OK and most() <= 128 << 20, (rows, n, cols)
""")
